"""The operators of a paged KV cache, and the verification of drafted tokens, as cases.

Attention of each sequence's newest tokens over a cache in pages; tokens written into the pages (bias, norms,
rotation, rounding) and read back; whole sequences read back; and drafted tokens judged by the target's and the
draft's probabilities with given random numbers. `run` computes them with elementary torch operations, or (`own`)
through the entry points of tokenstation5_amd.ts5hip. Head layouts, vocabularies and layer kinds are those of the
models in tokenstation5_amd/synth.py: the 8B (32/8 heads of 128, pairs rotated in place), the 48x5120 target (40/8 of
128) and the 0.5B draft (14/2 of 64), both with biases and halves rotated, and Gemma 3's layers (heads of 256, norms of
queries and keys, sliding windows).

A pool holds pages of `page` slots, each laid out as a cache of `page` slots: q8 (int8 values, an f16 scale per 32) or
f16, [page][KV head][slot][head_dim]. A sequence's pages lie anywhere in it; its table names them in order, -1 behind
the last. Cached keys lie around a direction of their page's own. `exact` computes the same outputs in float64, from
the definitions.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
KV_F16, KV_Q8 = 1, 2
F32, F16 = 0, 1
EPS = 1e-6
HEADS = {"8b": (32, 8, 128), "14b": (40, 8, 128), "draft": (14, 2, 64), "gemma": (8, 4, 256)}
HALVES = {"8b": False, "14b": True, "draft": True, "gemma": True}  # how dimensions pair up for the rotation
BIAS = {"14b", "draft"}
NORMS = {"gemma"}


def listed():
    return [
        # A draft model's decode step early in a conversation: the smallest call.
        dict(name="attend_draft_1x700_f16", op="attend", heads="draft", kv="f16", batch=1, new=1, keys=700, page=16,
             window=0),
        # A decode step of one long conversation: few rows, many keys.
        dict(name="attend_8b_1x32768_q8", op="attend", heads="8b", kv="q8", batch=1, new=1, keys=32768, page=64,
             window=0),
        # A decode step of 24 conversations between 500 and 16k keys: the largest.
        dict(name="attend_8b_24x16384_q8", op="attend", heads="8b", kv="q8", batch=24, new=1, keys=16384, page=64,
             window=0),
        # A sliding layer of eight Gemma 3 conversations.
        dict(name="attend_gemma_8x8192_f16", op="attend", heads="gemma", kv="f16", batch=8, new=1, keys=8192, page=32,
             window=1024),
        # Eight conversations' verify batches: the pending token and five drafts each.
        dict(name="attend_14b_8x6x8192_q8", op="attend", heads="14b", kv="q8", batch=8, new=6, keys=8192, page=128,
             window=0),
        # The new tokens of a decode step of 16 conversations, written and read back.
        dict(name="store_8b_16_q8", op="store", heads="8b", kv="q8", batch=16, tokens=16, keys=4096, page=64, pad=0),
        # Prompt chunks of three conversations in one call, padded by seven tokens.
        dict(name="store_14b_2041_q8", op="store", heads="14b", kv="q8", batch=3, tokens=2041, keys=4096, page=128, pad=7),
        # One layer of a 4k conversation read back to be saved.
        dict(name="read_8b_1x4100_q8", op="read", heads="8b", kv="q8", batch=1, keys=4100, page=64, out="f32"),
        # One layer of eight conversations of up to 16k tokens.
        dict(name="read_8b_8x16384_q8", op="read", heads="8b", kv="q8", batch=8, keys=16384, page=64, out="f16"),
        # One conversation's five drafts by prompt lookup: certain drafts, no draft logits.
        dict(name="verify_8b_1x5", op="verify", vocab=128256, ld=128256, batch=1, drafts=5, model=False),
        # Four conversations' seven drafts each by the 0.5B draft model.
        dict(name="verify_14b_4x7", op="verify", vocab=151936, ld=151936, batch=4, drafts=7, model=True),
        # Sixteen conversations, with room for fewer drafts in some.
        dict(name="verify_14b_16x7", op="verify", vocab=151936, ld=151936, batch=16, drafts=7, model=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "store", "read", "verify"])
    if op == "verify":
        c = dict(op=op, vocab=rng.choice([128256, 151936, _log(rng, 1000, 151936)]))
        c["ld"] = c["vocab"] + rng.choice([0, 0, rng.randint(1, 200)])
        c["batch"], c["drafts"] = rng.choice([1, _log(rng, 2, 16)]), rng.choice([1, rng.randint(2, 7), rng.randint(2, 7)])
        c["model"] = rng.random() < 0.6
        return c
    c = dict(op=op, heads=rng.choice(["8b", "8b", "14b", "draft", "gemma"]), kv=rng.choice(["q8", "q8", "f16"]))
    c["batch"] = rng.choice([1, _log(rng, 2, 16)])
    most = 16384 // (2 if c["heads"] == "gemma" or c["kv"] == "f16" else 1)
    c["page"] = rng.choice([16, 32, 64, 64, 128, 256])
    if op == "attend":
        c["new"] = rng.choice([1, 1, 1, rng.randint(2, 8)])
        c["keys"] = c["new"] + _log(rng, 20, most // (1 if c["new"] == 1 else 4))
        c["window"] = rng.choice([0, 0, 0, _log(rng, 64, 4096)])
    elif op == "store":
        c["tokens"] = c["batch"] * rng.choice([1, _log(rng, 1, 2000 // c["batch"])])
        c["keys"] = c["tokens"] + _log(rng, 16, 2000)
        c["pad"] = rng.choice([0, rng.randint(1, 9)])
    else:
        c["batch"], c["out"] = min(c["batch"], 6), rng.choice(["f32", "f16"])
        c["keys"] = _log(rng, 40, most // 2)
    return c


# ---- inputs --------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _ctx():
    """The program's context: one stream on the GPU."""
    from tokenstation5_amd import ts5hip
    return ts5hip.Context(0)


def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) % (1 << 62))
    return g


def _lengths(case):
    """Keys of each sequence: the first has them all, the others spread (by logarithm) down to a 32nd."""
    least = case.get("new", 1)
    return [max(least, int(round(case["keys"] * 2.0 ** (-5 * (b * 0.6180339887 % 1))))) for b in range(case["batch"])]


def _i32(rows):
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def _table(case, seed, lengths):
    """Each sequence's pages, drawn from a pool that has some to spare: ([sequence][page], pages of the pool)."""
    page = case["page"]
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + 3 + sum(need) // 16
    order = torch.randperm(pool, generator=_gen(seed, 3), device=DEV).to(torch.int32)
    table = torch.full((len(need), max(need) + 2), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def _rounded(x, kv):
    """x [..][head_dim] as a cache keeps it: (values, scales), scales None for f16."""
    if kv == "f16":
        return x.to(torch.float16), None
    rows = x.reshape(*x.shape[:-1], -1, 32)
    sc = (rows.abs().amax(-1) / 127).to(torch.float16)
    by = sc.float().unsqueeze(-1)
    q = torch.where(by > 0, torch.round(rows / by).clamp(-127, 127), torch.zeros_like(rows))
    return q.to(torch.int8).reshape(x.shape), sc


def _pool(case, seed, pool, which):
    """K (which 0) or V (1) of every page."""
    _, hkv, hd = HEADS[case["heads"]]
    g = _gen(seed, 10 + which)
    x = torch.randn(pool, hkv, case["page"], hd, generator=g, device=DEV)
    if which == 0:
        x = 0.8 * x + 0.6 * torch.randn(pool, hkv, 1, hd, generator=g, device=DEV)
    return _rounded(x, case["kv"])


def _rope_table(n_pos, hd):
    """(cos, sin) of every position and pair: [n_pos][head_dim / 2][2]."""
    inv = 500000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    a = torch.arange(n_pos, device=DEV, dtype=torch.float64).unsqueeze(1) * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _tokens(case, lengths):
    """(sequence, position) of the call's tokens: each sequence's newest ones, then the padding."""
    if case["op"] == "read":
        return [(b, p) for b, n in enumerate(lengths) for p in range(n)]
    per = [(case["tokens"] * (b + 1)) // case["batch"] - case["tokens"] * b // case["batch"] for b in range(case["batch"])]
    return [(b, n - m + i) for b, (n, m) in enumerate(zip(lengths, per)) for i in range(m)] + [(-1, 0)] * case["pad"]


def _verify_inputs(case, seed):
    b, t, v, ld = case["batch"], case["drafts"], case["vocab"], case["ld"]
    g = _gen(seed, 21)
    # A few tokens stand out of each row, as a trained model's do; the draft model agrees up to some noise.
    logits = 2.0 * torch.randn(b, t + 1, ld, generator=g, device=DEV)
    top = torch.randint(0, v, (b, t + 1, 12), generator=g, device=DEV)
    logits.scatter_add_(2, top, 8 + 3 * torch.randn(b, t + 1, 12, generator=g, device=DEV))
    temperature = 0.5 + 0.7 * torch.rand(b, generator=g, device=DEV)
    if b > 3:
        temperature[3] = 0.0  # a conversation that takes the best token
    s = dict(logits=logits, temperature=temperature, draft_logits=None)
    by = temperature.clamp(min=0.1).view(b, 1, 1)
    if case["model"]:
        s["draft_logits"] = logits[:, :t] + 0.7 * torch.randn(b, t, ld, generator=g, device=DEV)
        from_rows = s["draft_logits"]
    else:
        from_rows = logits[:, :t]
    noise = torch.rand(b, t, v, generator=g, device=DEV).clamp(min=1e-9)
    s["drafts"] = (from_rows[:, :, :v] / by - torch.log(-torch.log(noise))).argmax(-1).to(torch.int32)
    s["n_draft"] = _i32([t - (i % 3 if i % 4 == 2 else 0) if t > 2 else t for i in range(b)])
    s["uniform"] = torch.rand(b, t + 1, generator=g, device=DEV)
    s["tokens"] = torch.zeros(b, t + 1, dtype=torch.int32, device=DEV)
    s["n_tokens"] = torch.zeros(b, dtype=torch.int32, device=DEV)
    s["logp"] = torch.zeros(b, t + 1, device=DEV)
    return s


def prepare(case, seed):
    s = dict(case)
    if case["op"] == "verify":
        s.update(_verify_inputs(case, seed))
    else:
        h, hkv, hd = HEADS[case["heads"]]
        lengths = _lengths(case)
        if case["op"] == "store":
            lengths = [max(n, -(-case["tokens"] // case["batch"])) for n in lengths]
        s.update(n_head=h, n_head_kv=hkv, head_dim=hd, lengths=lengths, scale=1.0 / math.sqrt(hd))
        s["table"], s["n_pages"] = _table(case, seed, lengths)
        for which, name in enumerate("kv"):
            s[name], s[name + "s"] = _pool(case, seed, s["n_pages"], which)
        g = _gen(seed, 1)
        if case["op"] == "attend":
            s["n_keys"] = _i32(lengths)
            s["q"] = torch.randn(case["batch"], case["new"], h * hd, generator=g, device=DEV)
            s["out"] = torch.zeros_like(s["q"])
        else:
            seq, pos = zip(*_tokens(case, lengths))
            s["seq"], s["pos"], s["ntok"] = _i32(seq), _i32(pos), len(seq)
            s["placed"] = torch.nonzero(s["seq"] >= 0).squeeze(1)
            kind = torch.float32 if case.get("out") == "f32" else torch.float16
            s["k_out"] = torch.zeros(len(seq), hkv * hd, dtype=kind, device=DEV)
            s["v_out"] = torch.zeros_like(s["k_out"])
        if case["op"] == "store":
            s["qkv"] = torch.randn(s["ntok"], (h + 2 * hkv) * hd, generator=g, device=DEV)
            s["bias"] = 0.5 * torch.randn((h + 2 * hkv) * hd, generator=g, device=DEV) if case["heads"] in BIAS else None
            for n in ("q_norm", "k_norm"):
                s[n] = 1 + 0.1 * torch.randn(hd, generator=g, device=DEV) if case["heads"] in NORMS else None
            s["n_pos"] = max(lengths) + 1
            s["rope"] = _rope_table(s["n_pos"], hd)
            s["q_out"] = torch.zeros(s["ntok"], h * hd, device=DEV)
    if own:
        s["ctx"] = _ctx()
        s["ctx"].sync()
    if DEV == "cuda":
        torch.cuda.synchronize()
    return s


# ---- one pass through the framework's entry points -------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(s):
    c, op = s["ctx"], s["op"]
    if op == "verify":
        c.verify_drafts(_ptr(s["logits"]), s["ld"], _ptr(s["draft_logits"]), s["ld"], s["vocab"], *s["drafts"].shape,
                        _ptr(s["drafts"]), _ptr(s["n_draft"]), _ptr(s["temperature"]), _ptr(s["uniform"]),
                        _ptr(s["tokens"]), _ptr(s["n_tokens"]), _ptr(s["logp"]))
        return s["tokens"], s["n_tokens"], s["logp"]
    h, hkv, hd = s["n_head"], s["n_head_kv"], s["head_dim"]
    pool = (KV_Q8 if s["kv"] == "q8" else KV_F16, _ptr(s["k"]), _ptr(s["ks"]), _ptr(s["v"]), _ptr(s["vs"]), s["n_pages"],
            s["page"], _ptr(s["table"]))
    if op == "attend":
        c.attn_paged(_ptr(s["q"]), s["batch"], s["new"], h, hkv, hd, *pool, s["table"].shape[1], _ptr(s["n_keys"]),
                     s["window"], s["scale"], _ptr(s["out"]))
        return s["out"]
    seqs = s["table"].shape
    if op == "store":
        c.rope_kv_append_paged(_ptr(s["qkv"]), s["ntok"], _ptr(s["seq"]), _ptr(s["pos"]), h, hkv, hd, hd,
                               HALVES[s["heads"]], _ptr(s["rope"]), s["n_pos"], _ptr(s["q_out"]), *pool, *seqs,
                               bias=_ptr(s["bias"]), q_norm=_ptr(s["q_norm"]), k_norm=_ptr(s["k_norm"]), eps=EPS)
    c.kv_read_paged(s["ntok"], _ptr(s["seq"]), _ptr(s["pos"]), hkv, hd, *pool, *seqs,
                    F32 if s.get("out") == "f32" else F16, _ptr(s["k_out"]), _ptr(s["v_out"]))
    return (s["q_out"], s["k_out"], s["v_out"]) if op == "store" else (s["k_out"], s["v_out"])


# ---- the same in elementary torch operations, in float32 -------------------------------------------

def _values(x, sc):
    """Cached values in float32."""
    if sc is None:
        return x.float()
    return (x.reshape(*sc.shape, 32).float() * sc.float().unsqueeze(-1)).reshape(x.shape)


def _attend(s):
    b, new, h, hkv, hd = s["batch"], s["new"], s["n_head"], s["n_head_kv"], s["head_dim"]
    pages = s["table"].long().clamp(min=0)
    n = pages.shape[1] * s["page"]

    def all_keys(which):  # [sequence][KV head][key][head_dim]
        x = _values(s[which][pages], None if s[which + "s"] is None else s[which + "s"][pages])
        return x.permute(0, 2, 1, 3, 4).reshape(b, hkv, n, hd)

    q = s["q"].reshape(b, new, hkv, h // hkv, hd).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, hd)
    scores = (q @ all_keys("k").transpose(2, 3) * s["scale"]).reshape(b, hkv, h // hkv, new, n)
    key = torch.arange(n, device=q.device)
    end = s["n_keys"].view(b, 1) - new + 1 + torch.arange(new, device=q.device)  # past each query's own key
    seen = key < end.unsqueeze(2)
    if s["window"]:
        seen &= key >= (end - s["window"]).unsqueeze(2)
    scores = torch.where(seen.view(b, 1, 1, new, n), scores, torch.full_like(scores, -math.inf))
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    w = (w / w.sum(-1, keepdim=True)).reshape(b, hkv, -1, n)
    # (keys that no query sees may be anything, a pool's rows of other sequences among them)
    out = w @ torch.where(seen.any(1).view(b, 1, n, 1), all_keys("v"), torch.zeros((), device=q.device))
    return out.reshape(b, hkv, h // hkv, new, hd).permute(0, 3, 1, 2, 4).reshape(b, new, -1)


def _rotated(x, cs, halves):
    """x [token][head][head_dim] by (cos, sin) [token][head_dim / 2][2]."""
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    half = x.shape[-1] // 2
    x0, x1 = (x[..., :half], x[..., half:]) if halves else (x[..., 0::2], x[..., 1::2])
    y0, y1 = x0 * c - x1 * sn, x0 * sn + x1 * c
    return torch.cat([y0, y1], -1) if halves else torch.stack([y0, y1], -1).reshape(x.shape)


def _places(s):
    """(tokens that have a place, their pages, their slots)."""
    at = s["placed"]
    pos = s["pos"][at].long()
    return at, s["table"][s["seq"][at].long(), pos // s["page"]].long(), pos % s["page"]


def _read(s):
    at, page, slot = _places(s)
    outs = []
    for which in "kv":
        got = _values(s[which][page, :, slot], None if s[which + "s"] is None else s[which + "s"][page, :, slot])
        out = torch.zeros_like(s[which + "_out"])
        out[at] = got.reshape(len(at), -1).to(out.dtype)
        outs.append(out)
    return outs


def _store(s):
    h, hkv, hd = s["n_head"], s["n_head_kv"], s["head_dim"]
    at, page, slot = _places(s)
    x = s["qkv"][at] if s["bias"] is None else s["qkv"][at] + s["bias"]
    q, k, v = x.reshape(len(at), -1, hd).split([h, hkv, hkv], 1)
    cs = s["rope"][s["pos"][at].long()]
    parts = []
    for y, w in ((q, s["q_norm"]), (k, s["k_norm"])):
        if w is not None:
            y = y * (1 / torch.sqrt((y * y).sum(-1, keepdim=True) / hd + EPS)) * w
        parts.append(_rotated(y, cs, HALVES[s["heads"]]))
    q_out = torch.zeros_like(s["q_out"])
    q_out[at] = parts[0].reshape(len(at), -1)
    for which, y in (("k", parts[1]), ("v", v)):
        values, scales = _rounded(y, s["kv"])
        s[which][page, :, slot] = values
        if scales is not None:
            s[which + "s"][page, :, slot] = scales
    return q_out, *_read(s)


def _weights(logits, temperature, v):
    """Probabilities of each row's first v entries at its sequence's temperature, in float64; at 0 all of it is at
    the first of the largest entries."""
    x = logits[:, :, :v].double()
    top = x.amax(-1, keepdim=True)
    t = temperature.double().view(-1, 1, 1)
    index = torch.arange(v, device=x.device)
    best = torch.where(x == top, index, torch.full_like(index, v)).amin(-1, keepdim=True)
    w = torch.where(t > 0, torch.exp((x - top) / torch.where(t > 0, t, torch.ones_like(t))), (index == best).double())
    return w / w.sum(-1, keepdim=True)


def _verify(s):
    # (64 bits: a token is the first whose cumulative weight passes a bound)
    v, n = s["vocab"], s["drafts"].shape[1]
    p = _weights(s["logits"], s["temperature"], v)
    b = p.shape[0]
    drafts = s["drafts"].long()
    rows = torch.arange(b, device=p.device)
    certain = torch.zeros(b, n, v, dtype=torch.float64, device=p.device).scatter_(2, drafts.unsqueeze(2), 1.0)
    if s["draft_logits"] is None:
        q = certain
    else:
        greedy = (s["temperature"] <= 0).view(b, 1, 1)  # (the best token counts, whatever the draft's probabilities)
        q = torch.where(greedy, certain, _weights(s["draft_logits"], s["temperature"], v))
    pd, qd = (x[:, :n].gather(2, drafts.unsqueeze(2)).squeeze(2) for x in (p, q))
    kept = (s["uniform"][:, :n].double() * qd < pd) & (torch.arange(n, device=p.device) < s["n_draft"].view(b, 1))
    m = kept.to(torch.int64).cumprod(1).sum(1)
    row = p[rows, m]
    left = torch.where((m < s["n_draft"]).view(b, 1), row - q[rows, m.clamp(max=n - 1)], row).clamp(min=0)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, row)
    cum = left.cumsum(1)
    drawn = (cum <= s["uniform"][:, n:].double() * cum[:, -1:]).sum(1)
    place = torch.arange(n + 1, device=p.device)
    tokens = torch.cat([drafts, drafts[:, :1]], 1)
    tokens = torch.where(place == m.view(b, 1), drawn.view(b, 1), tokens)
    logp = torch.log(p.gather(2, tokens.unsqueeze(2)).squeeze(2)).float()
    behind = place > m.view(b, 1)
    tokens = torch.where(behind, torch.full_like(tokens, -1), tokens)
    return tokens.to(torch.int32), (m + 1).to(torch.int32), torch.where(behind, torch.zeros_like(logp), logp)


def run(s):
    if own:
        return _run_own(s)
    return {"attend": _attend, "store": _store, "read": lambda x: tuple(_read(x)), "verify": _verify}[s["op"]](s)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "verify":
        rows = case["batch"] * (case["drafts"] + 1 + (case["drafts"] if case["model"] else 0))
        return {"bytes": 4 * rows * case["vocab"] + 20 * case["batch"] * (case["drafts"] + 1), "flops": 20 * rows * case["vocab"]}
    h, hkv, hd = HEADS[case["heads"]]
    one = hkv * (hd * 2 if case["kv"] == "f16" else hd + hd // 32 * 2)  # a key (or a value) of every KV head
    lengths = _lengths(case)
    if op == "attend":
        new, win = case["new"], case["window"] or 1 << 30
        read = sum(min(n, win + new - 1) for n in lengths)
        pairs = sum(min(n - new + t + 1, win) for n in lengths for t in range(new))
        return {"bytes": 2 * one * read + case["batch"] * new * 8 * h * hd, "flops": 4 * hd * h * pairs}
    if op == "store":
        n = case["tokens"]
        return {"bytes": n * (4 * (2 * h + 2 * hkv) * hd + 2 * one + 4 * hkv * hd), "flops": 10 * n * (h + 2 * hkv) * hd}
    n = sum(lengths)
    return {"bytes": n * (2 * one + 2 * hkv * hd * (4 if case["out"] == "f32" else 2)), "flops": 2 * n * hkv * hd}


# ---- the definitions in float64 --------------------------------------------------------------------

def _exact_row(s, which, b, h, n):
    """The first n keys (or values) of KV head h of sequence b."""
    pages = s["table"][b, :-(-n // s["page"])].long()
    x = s[which][pages, h].double().flatten(0, 1)[:n]
    if s[which + "s"] is not None:
        x = x * s[which + "s"][pages, h].double().flatten(0, 1)[:n].repeat_interleave(32, dim=1)
    return x


def _exact_attend(s):
    H, hkv, hd, new = s["n_head"], s["n_head_kv"], s["head_dim"], s["new"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(s["lengths"]):
        for h in range(hkv):
            k, v = (_exact_row(s, m, b, h, n) for m in "kv")
            for t in range(new):
                end = n - new + t + 1
                first = max(0, end - s["window"]) if s["window"] else 0
                for j in range(h * (H // hkv), (h + 1) * (H // hkv)):
                    e = (k[first:end] * s["q"][b, t, j * hd:(j + 1) * hd].double()).sum(1) * s["scale"]
                    p = (e - e.max()).exp()
                    out[b, t, j * hd:(j + 1) * hd] = (v[first:end] * p.unsqueeze(1)).sum(0) / p.sum()
    return out


def _exact_cached(y, kv):
    """y (float64) as a cache keeps it."""
    if kv == "f16":
        return y.to(torch.float16).double()
    g = y.reshape(*y.shape[:-1], -1, 32)
    sc = (g.abs().max(-1, keepdim=True).values / 127.0).to(torch.float16).double()
    q = (g / torch.where(sc > 0, sc, torch.ones_like(sc))).round().clamp(-127, 127)
    return (q * sc).reshape(y.shape)


def _exact_store(s):
    h, hkv, hd = s["n_head"], s["n_head_kv"], s["head_dim"]
    x = s["qkv"].double() + (0 if s["bias"] is None else s["bias"].double())
    x = x.reshape(s["ntok"], h + 2 * hkv, hd)
    has = (s["seq"] >= 0).view(-1, 1, 1)
    turn = torch.view_as_complex(s["rope"][s["pos"].long()].double()).unsqueeze(1)

    def turned(y, w):
        if w is not None:
            y = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
        if HALVES[s["heads"]]:
            y = torch.stack([y[..., :hd // 2], y[..., hd // 2:]], -1)
        else:
            y = y.reshape(*y.shape[:-1], hd // 2, 2)
        z = torch.view_as_real(torch.view_as_complex(y.contiguous()) * turn)
        return torch.cat([z[..., 0], z[..., 1]], -1) if HALVES[s["heads"]] else z.flatten(-2)

    q, k, v = turned(x[:, :h], s["q_norm"]), turned(x[:, h:h + hkv], s["k_norm"]), x[:, h + hkv:]
    outs = (q, _exact_cached(k, s["kv"]), _exact_cached(v, s["kv"]))
    return tuple(torch.where(has, o, torch.zeros_like(o)).flatten(1) for o in outs)


def _exact_read(s):
    outs = []
    for which in "kv":
        rows = [torch.stack([_exact_row(s, which, b, h, n) for h in range(s["n_head_kv"])], 1).flatten(1)
                for b, n in enumerate(s["lengths"])]
        outs.append(torch.cat(rows))
    return tuple(outs)


def _exact_verify(s):
    b, n, v = s["batch"], s["drafts"].shape[1], s["vocab"]
    tokens, counts = torch.full((b, n + 1), -1, dtype=torch.int32), []
    logp = torch.zeros(b, n + 1, dtype=torch.float64)
    for i in range(b):
        t, u = float(s["temperature"][i]), s["uniform"][i].double().tolist()

        def log_rows(x):
            return torch.log_softmax(x[:v].double() / t, 0)

        m, end = 0, int(s["n_draft"][i])
        while True:
            row, d = s["logits"][i, m], int(s["drafts"][i, m]) if m < end else -1
            if t <= 0:
                best = int(torch.nonzero(row[:v] == row[:v].max())[0])
                tokens[i, m] = best
                if d != best:
                    break
                m += 1
                continue
            lp = log_rows(row)
            p = lp.exp()
            q = None
            if d >= 0:
                q = torch.zeros_like(p)
                q[d] = 1.0
                if s["draft_logits"] is not None:
                    q = log_rows(s["draft_logits"][i, m]).exp()
                if u[m] * float(q[d]) < float(p[d]):
                    tokens[i, m], logp[i, m] = d, lp[d]
                    m += 1
                    continue
            w = p if q is None else torch.relu(p - q)
            c = torch.cumsum(w, 0)
            at = int(torch.searchsorted(c, torch.tensor([u[n] * float(c[-1])], dtype=c.dtype, device=c.device), right=True))
            tokens[i, m], logp[i, m] = at, lp[at]
            break
        counts.append(m + 1)
    return tokens, torch.tensor(counts, dtype=torch.int32), logp


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "store": _exact_store, "read": _exact_read, "verify": _exact_verify}[case["op"]](s)
