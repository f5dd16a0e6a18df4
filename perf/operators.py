"""The operators around a KV cache that a long conversation and tree speculation need, as cases.

Attention of a tree of drafted tokens; attention that adds each key's weight to a running sum (decode steps
and prompt chunks); eviction of the keys with the least weight; the bounds of the keys of every block of a
cache; and attention over the blocks that those bounds pick for each query. `run` computes them with
elementary torch operations, or (`own`) through the entry points of tokenstation5_amd.ts5hip. Head layouts
are those of the models in tokenstation5_amd/synth.py: the 8B (32/8 heads of 128), the 48x5120 target
(40/8 of 128), the 0.5B draft (14/2 of 64) and Gemma 3's heads of 256.

Caches are q8 (int8 values, an f16 scale per 32) or f16, [sequence][KV head][slot][head_dim]; queries and
cached keys and values are normally distributed, the keys around a direction that changes every 128 keys.
`exact` computes the same outputs in float64, from the definitions.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
KV_F16, KV_Q8 = 1, 2
HEADS = {"8b": (32, 8, 128), "14b": (40, 8, 128), "draft": (14, 2, 64), "gemma": (8, 4, 256)}


def listed():
    return [
        # A draft model's own tree of 7 continuations early in a conversation: the smallest call.
        dict(name="tree_draft_7x700_f16", op="tree", heads="draft", kv="f16", batch=1, tree=7, keys=700),
        # The 8B verifies a tree of 21 drafts in a 4k conversation.
        dict(name="tree_8b_21x4096_q8", op="tree", heads="8b", kv="q8", batch=1, tree=21, keys=4096),
        # Four conversations of up to 8k, each with the largest tree.
        dict(name="tree_8b_4x64x8192_q8", op="tree", heads="8b", kv="q8", batch=4, tree=64, keys=8192),
        # A decode step of the draft model that keeps count of its keys' weights.
        dict(name="weights_draft_1x1500_f16", op="weights", heads="draft", kv="f16", batch=1, keys=1500),
        # A decode step of 16 conversations of up to 16k keys.
        dict(name="weights_8b_16x16384_q8", op="weights", heads="8b", kv="q8", batch=16, keys=16384),
        # A prompt chunk of the 8B at the end of 4k keys, its weights counted.
        dict(name="weights_prompt_256x4096_q8", op="prompt", heads="8b", kv="q8", batch=256, keys=4096),
        # One layer of a 4k conversation cut back to 2048 keys.
        dict(name="evict_8b_1x4100_q8", op="evict", heads="8b", kv="q8", batch=1, keys=4100, keep=2048),
        # Eight conversations of up to 32k keys cut back to 8k.
        dict(name="evict_8b_8x32768_q8", op="evict", heads="8b", kv="q8", batch=8, keys=32768, keep=8192),
        # A decode step that completes a block of 64 keys.
        dict(name="bounds_8b_1x64_q8", op="bounds", heads="8b", kv="q8", batch=1, keys=4096, new=64, block=64),
        # The whole caches of four 16k prompts on the 48x5120 target.
        dict(name="bounds_14b_4x16384_f16", op="bounds", heads="14b", kv="f16", batch=4, keys=16384, new=16384,
             block=64),
        # A decode step of one 32k conversation that reads 32 of its 512 blocks.
        dict(name="sparse_8b_1x32768_q8", op="sparse", heads="8b", kv="q8", batch=1, keys=32768, block=64, pick=32),
        # A decode step of 16 conversations of up to 32k keys, 128 blocks of 32 keys each.
        dict(name="sparse_8b_16x32768_q8", op="sparse", heads="8b", kv="q8", batch=16, keys=32768, block=32, pick=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "weights", "prompt", "evict", "bounds", "sparse"])
    heads = rng.choice(["8b", "8b", "14b", "draft", "gemma"])
    c = dict(op=op, heads=heads, kv=rng.choice(["q8", "f16"]))
    if op == "tree":
        c["batch"] = rng.choice([1, 1, rng.randint(2, 3)])
        c["tree"] = rng.choice([1, _log(rng, 2, 16), rng.randint(17, 64)])
        c["keys"] = _log(rng, 64, 8192)
    elif op == "weights":
        c["batch"] = rng.choice([1, rng.randint(2, 12)])
        c["keys"] = _log(rng, 32, 16384 // (2 if heads == "gemma" or c["kv"] == "f16" else 1))
    elif op == "prompt":
        c["batch"] = rng.choice([1, _log(rng, 2, 200)])
        c["keys"] = c["batch"] + _log(rng, 16, 3600)
    elif op == "evict":
        c["batch"] = rng.choice([1, rng.randint(2, 6)])
        c["keys"] = _log(rng, 300, 16384)
        c["keep"] = rng.randint(128, max(129, c["keys"] // 2))
    else:
        c["batch"] = rng.choice([1, rng.randint(2, 8 if op == "sparse" else 3)])
        c["block"] = rng.choice([16, 32, 64, 128])
        c["keys"] = _log(rng, 256, 16384)
        if op == "bounds":
            c["new"] = rng.choice([1, rng.randint(2, 200), c["keys"]])
        else:
            c["pick"] = min(rng.choice([_log(rng, 4, 64), 32]), 4096 // c["block"])
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


def _slots(case):
    n = case["keys"] + (case["tree"] if case["op"] == "tree" else 0)
    return -(-n // 256) * 256


def _lengths(case):
    """Keys of each sequence: the first has them all, the others end earlier, up to a quarter."""
    return [case["keys"] - b * case["keys"] // (4 * case["batch"]) for b in range(case["batch"])]


def _seqs(case):
    return 1 if case["op"] == "prompt" else case["batch"]


def _cache(case, seed, b, which):
    """K (which 0) or V (1) of sequence b: (values, scales), scales None for f16."""
    _, hkv, hd = HEADS[case["heads"]]
    n, g = _slots(case), _gen(seed, 1000 + 2 * b + which)
    x = torch.randn(hkv, n, hd, generator=g, device=DEV)
    if which == 0:
        topics = torch.randn(hkv, -(-n // 128), hd, generator=g, device=DEV)
        x = 0.8 * x + 0.6 * topics.repeat_interleave(128, 1)[:, :n]
    if case["kv"] == "f16":
        return x.to(torch.float16), None
    rows = x.reshape(hkv, n, hd // 32, 32)
    sc = (rows.abs().amax(-1) / 127).to(torch.float16)
    q = torch.round(rows / sc.float().unsqueeze(-1)).clamp_(-127, 127)
    return q.to(torch.int8).reshape(x.shape), sc


def _queries(case, seed):
    h, _, hd = HEADS[case["heads"]]
    rows = case["batch"] * case.get("tree", 1)
    return torch.randn(rows, h * hd, generator=_gen(seed, 1), device=DEV)


def _tree_masks(case, seed):
    """Each drafted token's ancestors and itself as bits, from parents drawn among the tokens before it."""
    g = torch.Generator()
    g.manual_seed(int(seed) * 7919 + 5)
    out = []
    for _ in range(case["batch"]):
        m = []
        for t in range(case["tree"]):
            p = -1 if t == 0 else int(torch.randint(-1, t, (1,), generator=g)) if t < 4 else \
                int(torch.randint(t // 3, t, (1,), generator=g))
            m.append((m[p] if p >= 0 else 0) | 1 << t)
        out.append([v - (1 << 64) if v >= 1 << 63 else v for v in m])
    return torch.tensor(out, dtype=torch.int64, device=DEV)


def _sums(case, seed):
    """Weights accumulated so far: long-tailed, none at all for some keys."""
    _, hkv, _ = HEADS[case["heads"]]
    x = torch.randn(_seqs(case), hkv, _slots(case), generator=_gen(seed, 7), device=DEV)
    return torch.where(x < -1.5, torch.zeros_like(x), torch.exp(1.5 * x))


def _first_last(case):
    """Keys that eviction keeps in any case: the first ones and the most recent ones."""
    return min(4, case["keep"] // 4), min(64, case["keep"] // 4)


def _bounds_of(k, ks, n, block):
    """Lowest and highest value of every dimension over each block of the first n slots: f16, lowest rounded
    down and highest rounded up, [KV head][block][2][head_dim]; blocks past n are zero."""
    hkv, slots, hd = k.shape
    x = k.float() if ks is None else (k.reshape(hkv, slots, -1, 32).float() * ks.float().unsqueeze(-1)).reshape(k.shape)
    nb, used = -(-slots // block), -(-n // block)
    out = torch.zeros(hkv, nb, 2, hd, dtype=torch.float16, device=k.device)
    pad = used * block - n
    for which, fill in ((0, math.inf), (1, -math.inf)):
        y = torch.cat([x[:, :n], torch.full((hkv, pad, hd), fill, device=k.device)], 1) if pad else x[:, :n]
        y = y.reshape(hkv, used, block, hd)
        v = y.amin(2) if which == 0 else y.amax(2)
        out[:, :used, which] = _round_to_f16(v, up=which == 1)
    return out


def _round_to_f16(v, up):
    """v (float32) as the nearest f16 that is not above (or, up, not below) it."""
    h = v.to(torch.float16)
    wrong = h.float() < v if up else h.float() > v
    bits = h.view(torch.int16).to(torch.int32) & 0xFFFF
    away = (bits & 0x8000 == 0) == up  # the step goes away from zero
    step = torch.where(away, bits + 1, bits - 1)
    step = torch.where(bits & 0x7FFF == 0, torch.full_like(bits, 0x0001 if up else 0x8001), step)
    bits = torch.where(wrong, step, bits)
    return torch.where(bits >= 0x8000, bits - 0x10000, bits).to(torch.int16).view(torch.float16)


def prepare(case, seed):
    op = case["op"]
    h, hkv, hd = HEADS[case["heads"]]
    s = dict(case, n_head=h, n_head_kv=hkv, head_dim=hd, n_ctx=_slots(case), scale=1.0 / math.sqrt(hd))
    kv = [[_cache(case, seed, b, which) for b in range(_seqs(case))] for which in ((0,) if op == "bounds" else (0, 1))]
    for name, seqs in zip("kv", kv):
        s[name] = torch.stack([v for v, _ in seqs])
        s[name + "s"] = torch.stack([sc for _, sc in seqs]) if case["kv"] == "q8" else None
    s["lengths"] = [case["keys"]] if op == "prompt" else _lengths(case)
    s["n_keys"] = torch.tensor(s["lengths"], dtype=torch.int32, device=DEV)
    if op not in ("evict", "bounds"):
        s["q"] = _queries(case, seed)
        s["out"] = torch.zeros_like(s["q"])
    if op == "tree":
        s["mask"] = _tree_masks(case, seed)
    elif op in ("weights", "prompt"):
        s["acc"] = _sums(case, seed)
        s["acc_out"] = torch.zeros_like(s["acc"])
    elif op == "evict":
        keep, b = case["keep"], case["batch"]
        s["acc"] = _sums(case, seed)
        s["slots_out"] = -(-keep // 256) * 256
        for n in "kv":
            s[n + "_out"] = torch.zeros(b, hkv, s["slots_out"], hd, dtype=s[n].dtype, device=DEV)
            s[n + "s_out"] = None if s[n + "s"] is None else \
                torch.zeros(b, hkv, s["slots_out"], hd // 32, dtype=torch.float16, device=DEV)
        s["acc_out"] = torch.zeros(b, hkv, s["slots_out"], device=DEV)
        s["kept"] = torch.zeros(b, hkv, keep, dtype=torch.int32, device=DEV)
        s["n_out"] = torch.zeros(b, dtype=torch.int32, device=DEV)
    elif op == "bounds":
        s["bounds"] = torch.zeros(case["batch"], hkv, -(-s["n_ctx"] // case["block"]), 2, hd, dtype=torch.float16,
                                  device=DEV)
    elif op == "sparse":
        s["bounds"] = torch.stack([_bounds_of(s["k"][b], None if s["ks"] is None else s["ks"][b], n, case["block"])
                                   for b, n in enumerate(s["lengths"])])
        s["picked"] = torch.zeros(case["batch"], hkv, case["pick"], dtype=torch.int32, device=DEV)
    if own:
        s["ctx"] = _ctx()
        s["kv_type"] = KV_Q8 if case["kv"] == "q8" else KV_F16
        s["ctx"].sync()
    if DEV == "cuda":
        torch.cuda.synchronize()
    return s


# ---- one pass through the framework's entry points -------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(s):
    c, op, b = s["ctx"], s["op"], s["batch"]
    heads = s["n_head"], s["n_head_kv"], s["head_dim"]
    kv = s["kv_type"], _ptr(s["k"]), _ptr(s["ks"])
    if op != "bounds":
        kv += _ptr(s["v"]), _ptr(s["vs"])
    n_keys = _ptr(s["n_keys"])
    if op == "tree":
        c.attn_tree(_ptr(s["q"]), b, s["tree"], *heads, *kv, s["n_ctx"], n_keys, _ptr(s["mask"]), s["scale"],
                    _ptr(s["out"]))
        return s["out"]
    if op == "weights":
        c.attn_decode_weights(_ptr(s["q"]), b, *heads, *kv, s["n_ctx"], n_keys, s["scale"], _ptr(s["out"]),
                              _ptr(s["acc"]), _ptr(s["acc_out"]))
        return s["out"], s["acc_out"]
    if op == "prompt":
        c.attn_prompt_weights(_ptr(s["q"]), b, *heads, *kv, s["n_ctx"], s["keys"] - b, s["scale"], _ptr(s["out"]),
                              _ptr(s["acc"]), _ptr(s["acc_out"]))
        return s["out"], s["acc_out"]
    if op == "evict":
        c.kv_evict(b, *heads[1:], *kv, s["n_ctx"], n_keys, _ptr(s["acc"]), s["keep"], *_first_last(s),
                   s["slots_out"], _ptr(s["k_out"]), _ptr(s["ks_out"]), _ptr(s["v_out"]), _ptr(s["vs_out"]),
                   _ptr(s["acc_out"]), _ptr(s["kept"]), _ptr(s["n_out"]))
        return [s[n] for n in ("k_out", "ks_out", "v_out", "vs_out", "acc_out", "kept", "n_out")]
    if op == "bounds":
        c.kv_block_bounds(b, *heads[1:], *kv, s["n_ctx"], n_keys, s["new"], s["block"], _ptr(s["bounds"]))
        return s["bounds"]
    c.attn_sparse(_ptr(s["q"]), b, *heads, *kv, s["n_ctx"], n_keys, 1, _ptr(s["bounds"]), s["block"], s["pick"],
                  s["scale"], _ptr(s["out"]), _ptr(s["picked"]))
    return s["out"], s["picked"]


# ---- the same in elementary torch operations, in float32 -------------------------------------------

def _values(s, which, b, n):
    """K or V of sequence b's first n keys in float32: [KV head][n][head_dim]."""
    x = s[which][b, :, :n].float()
    if s[which + "s"] is None:
        return x
    sc = s[which + "s"][b, :, :n].float()
    return (x.reshape(*sc.shape, 32) * sc.unsqueeze(-1)).reshape(x.shape)


def _softmax(scores):
    """Weights of the last axis; a row with no key (all -inf) has none."""
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    return p / torch.where(l == 0, torch.ones_like(l), l)


def _grouped(q, hkv, hd):
    """Query rows [rows][H HD] as [KV head][rows * G][head_dim]."""
    rows = q.shape[0]
    return q.reshape(rows, hkv, -1, hd).permute(1, 0, 2, 3).reshape(hkv, -1, hd)


def _ungrouped(o, rows):
    hkv, rg, hd = o.shape
    return o.reshape(hkv, rows, rg // rows, hd).permute(1, 0, 2, 3).reshape(rows, -1)


def _attend(s, q, b, n, seen=None):
    """Queries [rows][H HD] over sequence b's first n keys; seen [rows][n] or None: (outputs, weights [KV
    head][rows * G][n])."""
    hkv, hd = s["n_head_kv"], s["head_dim"]
    qg = _grouped(q, hkv, hd)
    scores = qg @ _values(s, "k", b, n).transpose(1, 2) * s["scale"]
    if seen is not None:
        scores = torch.where(seen.repeat_interleave(qg.shape[1] // q.shape[0], 0), scores,
                             torch.full_like(scores, -math.inf))
    w = _softmax(scores)
    return _ungrouped(w @ _values(s, "v", b, n), q.shape[0]), w


def _tree_seen(mask, n, tree):
    """[tree][n + tree]: the past, and the drafted tokens whose bit is set."""
    bits = (mask.unsqueeze(1) >> torch.arange(tree, device=mask.device)) & 1
    return torch.cat([torch.ones(tree, n, dtype=torch.bool, device=mask.device), bits.bool()], 1)


def _causal_seen(nq, n, dev):
    return torch.arange(n, device=dev) <= torch.arange(n - nq, n, device=dev).unsqueeze(1)


def _evict_kept(sums, n, keep, first, last):
    """Slots kept of n, ascending: the first and last ones, then the largest sums, ties to the lowest slot."""
    x = sums[:, :n].clone()
    x[:, :first] = math.inf
    x[:, n - last:] = math.inf
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    return torch.sort(order[:, :min(keep, n)], dim=1)[0]


def _take(x, rows):
    """x [KV head][slot][...] at slots rows [KV head][m]."""
    return torch.stack([x[h, rows[h]] for h in range(x.shape[0])])


def _block_scores(q, bounds):
    """The highest score that a key inside a block's bounds can have with any of the KV head's queries, before
    the scale: q [KV head][G][head_dim], bounds [KV head][blocks][2][head_dim] -> [KV head][blocks], float64."""
    q, lo, hi = q.double().unsqueeze(2), bounds[:, :, 0].double().unsqueeze(1), bounds[:, :, 1].double().unsqueeze(1)
    return torch.where(q >= 0, q * hi, q * lo).sum(-1).amax(1)


def _pick(scores, pick):
    """Blocks read of [KV head][blocks], ascending: the last, the first, then the highest scores."""
    nb = scores.shape[1]
    x = scores.clone()
    x[:, 0] = math.inf
    order = torch.sort(x[:, :nb - 1], dim=1, descending=True, stable=True)[1][:, :pick - 1]
    last = torch.full_like(order[:, :1], nb - 1) if nb > 1 else torch.zeros(x.shape[0], 1, dtype=torch.int64, device=x.device)
    return torch.sort(torch.cat([order, last], 1), dim=1)[0]


def run(s):
    if own:
        return _run_own(s)
    op, hkv, hd = s["op"], s["n_head_kv"], s["head_dim"]
    if op == "tree":
        t = s["tree"]
        return torch.cat([_attend(s, s["q"][b * t:(b + 1) * t], b, n + t, _tree_seen(s["mask"][b], n, t))[0]
                          for b, n in enumerate(s["lengths"])])
    if op in ("weights", "prompt"):
        acc, outs = torch.zeros_like(s["acc"]), []
        for b, n in enumerate(s["lengths"]):
            q = s["q"] if op == "prompt" else s["q"][b:b + 1]
            o, w = _attend(s, q, b, n, _causal_seen(s["batch"], n, q.device) if op == "prompt" else None)
            outs.append(o)
            acc[b, :, :n] = s["acc"][b, :, :n] + w.sum(1)
        return torch.cat(outs), acc
    if op == "evict":
        out = {n: None if s[n] is None else torch.zeros_like(s[n])
               for n in ("k_out", "ks_out", "v_out", "vs_out", "acc_out")}
        kept = torch.full_like(s["kept"], -1)
        for b, n in enumerate(s["lengths"]):
            rows = _evict_kept(s["acc"][b], n, s["keep"], *_first_last(s))
            m = rows.shape[1]
            kept[b, :, :m] = rows.to(torch.int32)
            for name in ("k", "ks", "v", "vs", "acc"):
                if s[name] is not None:
                    out[name + "_out"][b, :, :m] = _take(s[name][b], rows)
        return [*out.values(), kept, torch.clamp(s["n_keys"], max=s["keep"])]
    if op == "bounds":
        out = torch.zeros_like(s["bounds"])
        for b, n in enumerate(s["lengths"]):
            first = max(n - s["new"], 0) // s["block"]
            at = first * s["block"]
            got = _bounds_of(s["k"][b, :, at:n], None if s["ks"] is None else s["ks"][b, :, at:n], n - at, s["block"])
            out[b, :, first:first + got.shape[1]] = got
        return out
    outs, picked = [], torch.full_like(s["picked"], -1)
    for b, n in enumerate(s["lengths"]):
        q, block = _grouped(s["q"][b:b + 1], hkv, hd), s["block"]
        blocks = _pick(_block_scores(q, s["bounds"][b, :, :-(-n // block)]), s["pick"])
        picked[b, :, :blocks.shape[1]] = blocks.to(torch.int32)
        rows = (blocks.unsqueeze(2) * block + torch.arange(block, device=q.device)).reshape(hkv, -1)
        inside, rows = rows < n, rows.clamp(max=n - 1)
        kv = {m: (_take(s[m][b], rows).float() if s[m + "s"] is None else
                  (_take(s[m][b], rows).float().reshape(hkv, -1, hd // 32, 32)
                   * _take(s[m + "s"][b], rows).float().unsqueeze(-1)).reshape(hkv, -1, hd)) for m in "kv"}
        scores = q @ kv["k"].transpose(1, 2) * s["scale"]
        w = _softmax(torch.where(inside.unsqueeze(1), scores, torch.full_like(scores, -math.inf)))
        outs.append(_ungrouped(w @ kv["v"], 1))
    return torch.cat(outs), picked


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    op = case["op"]
    h, hkv, hd = HEADS[case["heads"]]
    one = hkv * (hd * 2 if case["kv"] == "f16" else hd + hd // 32 * 2)  # a key (or a value) of every KV head
    lengths = [case["keys"]] if op == "prompt" else _lengths(case)
    keys = sum(lengths)
    if op == "tree":
        t = case["tree"]
        keys += t * case["batch"]
        return {"bytes": 2 * one * keys + case["batch"] * t * (8 * h * hd + 8),
                "flops": 4 * hd * h * t * sum(n + t / 4 for n in lengths)}
    if op == "weights":
        return {"bytes": 2 * one * keys + 8 * hkv * keys + 8 * case["batch"] * h * hd, "flops": 4 * hd * h * keys}
    if op == "prompt":
        nq = case["batch"]
        return {"bytes": 2 * one * keys + 8 * hkv * keys + 8 * nq * h * hd,
                "flops": 4 * hd * h * (nq * (keys - nq) + nq * (nq + 1) // 2)}
    if op == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        return {"bytes": 4 * one * kept + 4 * hkv * keys + 8 * hkv * kept, "flops": hkv * keys}
    if op == "bounds":
        new = sum(-(-min(case["new"], n) // case["block"]) for n in lengths)
        return {"bytes": one * min(new * case["block"], keys) + 4 * hkv * hd * new,
                "flops": 2 * hkv * hd * new * case["block"]}
    nb = sum(-(-n // case["block"]) for n in lengths)
    read = sum(min(n, case["pick"] * case["block"]) for n in lengths)
    return {"bytes": 4 * hkv * hd * nb + 2 * one * read + case["batch"] * (8 * h * hd + 4 * hkv * case["pick"]),
            "flops": 2 * h * hd * nb + 4 * hd * h * read}


# ---- the definitions in float64 --------------------------------------------------------------------

def _exact_kv(s, which, b, h):
    x = s[which][b, h].double()
    if s[which + "s"] is not None:
        x *= s[which + "s"][b, h].double().repeat_interleave(32, dim=-1)
    return x


def _exact_head(s, q, b, hh, slots):
    """One query head (rows [r][HD]) over the slots given per row (a bool [r][n]): outputs and weights."""
    g = s["n_head"] // s["n_head_kv"]
    n = slots.shape[1]
    k, v = (_exact_kv(s, m, b, hh // g)[:n] for m in "kv")
    e = torch.einsum("rd,nd->rn", q.double(), k) * s["scale"]
    e = e.masked_fill(~slots, -math.inf)
    top = e.max(1, keepdim=True).values
    p = torch.where(slots, (e - top).exp(), torch.zeros_like(e))
    p = p / p.sum(1, keepdim=True)
    return p @ v, p


def _exact_f16(x, up):
    """float64 x to the f16 grid, up or down."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -14)))
    step = torch.exp2(e - 10)
    y = (torch.ceil(x / step) if up else torch.floor(x / step)) * step
    return y.to(torch.float16)


def exact(case, seed):
    s = prepare(case, seed)
    op, H, hkv, hd, g = s["op"], s["n_head"], s["n_head_kv"], s["head_dim"], s["n_head"] // s["n_head_kv"]
    dev = s["k"].device
    if op == "bounds":
        out = torch.zeros_like(s["bounds"])
        for b, n in enumerate(s["lengths"]):
            for h in range(hkv):
                k = _exact_kv(s, "k", b, h)
                for blk in range(max(n - s["new"], 0) // s["block"], -(-n // s["block"])):
                    rows = k[blk * s["block"]:min(n, (blk + 1) * s["block"])]
                    out[b, h, blk, 0] = _exact_f16(rows.min(0).values, False)
                    out[b, h, blk, 1] = _exact_f16(rows.max(0).values, True)
        return out
    if op == "evict":
        first, last = _first_last(s)
        outs = [None if s[m] is None else torch.zeros_like(s[m]) for m in ("k_out", "ks_out", "v_out", "vs_out", "acc_out")]
        kept = torch.full_like(s["kept"], -1)
        for b, n in enumerate(s["lengths"]):
            for h in range(hkv):
                a = s["acc"][b, h, :n].tolist()
                order = sorted(range(n), key=lambda i: (not (i < first or i >= n - last), -a[i], i))
                rows = sorted(order[:s["keep"]])
                kept[b, h, :len(rows)] = torch.tensor(rows, dtype=torch.int32, device=dev)
                at = torch.tensor(rows, device=dev)
                for o, m in zip(outs, ("k", "ks", "v", "vs", "acc")):
                    if o is not None:
                        o[b, h, :len(rows)] = s[m][b, h].index_select(0, at)
        return [*outs, kept, torch.tensor([min(n, s["keep"]) for n in s["lengths"]], dtype=torch.int32, device=dev)]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    acc = None
    if op in ("weights", "prompt"):
        acc = torch.zeros(s["acc"].shape, dtype=torch.float64, device=dev)
    picked = torch.full_like(s["picked"], -1) if op == "sparse" else None
    rows = {"tree": s.get("tree"), "prompt": s["batch"]}.get(op, 1)
    for b, n in enumerate(s["lengths"]):
        if op == "tree":
            bits = s["mask"][b].tolist()
            slots = torch.ones(rows, n + rows, dtype=torch.bool)
            for t in range(rows):
                for j in range(rows):
                    slots[t, n + j] = bool(bits[t] >> j & 1)
            slots = slots.to(dev)
        elif op == "prompt":
            slots = torch.ones(rows, n, dtype=torch.bool, device=dev).tril(n - rows)
        else:
            slots = torch.ones(1, n, dtype=torch.bool, device=dev)
        for hh in range(H):
            q = s["q"][b * rows:(b + 1) * rows, hh * hd:(hh + 1) * hd]
            if op == "sparse":
                if hh % g == 0:
                    nb = -(-n // s["block"])
                    lo, hi = (s["bounds"][b, hh // g, :nb, i].double() for i in (0, 1))
                    best = None
                    for j in range(g):
                        qq = s["q"][b, (hh + j) * hd:(hh + j + 1) * hd].double()
                        u = torch.maximum(qq * lo, qq * hi).sum(1)
                        best = u if best is None else torch.maximum(best, u)
                    u = best.tolist()
                    order = sorted(range(nb), key=lambda i: (i != nb - 1, i != 0, -u[i], i))
                    blocks = sorted(order[:s["pick"]])
                    picked[b, hh // g, :len(blocks)] = torch.tensor(blocks, dtype=torch.int32, device=dev)
                    slots = torch.zeros(1, n, dtype=torch.bool, device=dev)
                    for i in blocks:
                        slots[0, i * s["block"]:(i + 1) * s["block"]] = True
            o, p = _exact_head(s, q, b, hh, slots)
            out[b * rows:(b + 1) * rows, hh * hd:(hh + 1) * hd] = o
            if acc is not None:
                acc[b, hh // g, :n] += p.sum(0) + (s["acc"][b, hh // g, :n].double() if hh % g == 0 else 0)
    return out if op == "tree" else (out, picked) if op == "sparse" else (out, acc)
