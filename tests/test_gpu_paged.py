"""A cache in pages (attention of the newest tokens, tokens written into it and read back), through the C ABI, against
float64 numpy. The tolerance of an attention output is derived in test_gpu_cache_ops.py; its core is the same."""
import numpy as np
import pytest

from test_gpu_cache_ops import HEADS, attend, check_rows
from tokenstation5_amd import ts5hip

pytestmark = pytest.mark.gpu
Q8, F16 = ts5hip.KV_Q8, ts5hip.KV_F16


@pytest.fixture(scope="module")
def ctx():
    c = ts5hip.Context(0)
    yield c
    c.close()


def rounded(x, kv):
    """x [..][HD] (float32) as a cache keeps it: (values, scales or None)."""
    if kv == F16:
        return x.astype(np.float16), None
    r = x.reshape(*x.shape[:-1], -1, 32)
    sc = (np.abs(r).max(-1) / np.float32(127)).astype(np.float16)
    by = sc.astype(np.float32)[..., None]
    q = np.where(by > 0, np.clip(np.rint(r / np.where(by > 0, by, 1)), -127, 127), 0)
    return q.astype(np.int8).reshape(x.shape), sc


class Pages:
    """A pool of random K and V in host and device memory and the tables of sequences of `lengths`; k, v their values."""

    def __init__(self, ctx, rng, kv, HKV, HD, page, lengths, spare=3, n_table=None, std=1.0):
        self.ctx, self.kv, self.HKV, self.HD, self.page, self.lengths = ctx, kv, HKV, HD, page, lengths
        need = [-(-max(n, 0) // page) for n in lengths]
        self.n_pages, self.n_table = sum(need) + spare, n_table or max(max(need), 1) + 1
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table, at = np.full((len(lengths), self.n_table), -1, np.int32), 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.raw = {}
        for n in "kv":
            x = rng.standard_normal((self.n_pages, HKV, page, HD)).astype(np.float32) * np.float32(std)
            self.raw[n], sc = rounded(x, kv)
            if sc is not None:
                self.raw[n + "s"] = sc
        self.send()

    def send(self):
        self.dev = {n: self.ctx.to_device(a) for n, a in self.raw.items()}
        self.table_dev = self.ctx.to_device(self.table)
        return self

    def fetch(self):
        return {n: d.download(self.raw[n].dtype, self.raw[n].shape) for n, d in self.dev.items()}

    @property
    def args(self):
        """kv type, k, ks, v, vs, pages, page, table as the entry points take them."""
        d = self.dev
        return self.kv, d["k"], d.get("ks"), d["v"], d.get("vs"), self.n_pages, self.page, self.table_dev

    def values(self, n, raw=None):
        raw = raw or self.raw
        with np.errstate(invalid="ignore"):
            x = raw[n].astype(np.float64)
            if self.kv == Q8:
                x = x * np.repeat(raw[n + "s"].astype(np.float64), 32, axis=-1)
        return x

    def rows(self, n, b, h, count, raw=None):
        """The first `count` keys (values) of sequence b and KV head h, and which of them have a page."""
        out, has = np.zeros((count, self.HD)), np.zeros(count, bool)
        raw = raw or self.raw
        for i in range(-(-count // self.page)):
            p = self.table[b, i] if i < self.n_table else -1
            if 0 <= p < self.n_pages:
                m = min(self.page, count - i * self.page)
                x = raw[n][p, h, :m].astype(np.float64)
                if self.kv == Q8:
                    with np.errstate(invalid="ignore"):
                        x = x * np.repeat(raw[n + "s"][p, h, :m].astype(np.float64), 32, axis=-1)
                out[i * self.page:i * self.page + m], has[i * self.page:i * self.page + m] = x, True
        return out, has


def seen_by(n, T, window, has):
    """[T][n]: the keys that each of the T newest tokens reads."""
    key, end = np.arange(n)[None], n - T + 1 + np.arange(T)[:, None]
    return (key < end) & (key >= (end - window if window else 0)) & has[None]


def run_attn(ctx, c, q, n_keys, window, scale, H, out=None):
    B, T = q.shape[:2]
    out = out or ctx.alloc(q.nbytes)
    ctx.attn_paged(ctx.to_device(q), B, T, H, c.HKV, c.HD, *c.args, c.n_table, ctx.to_device(np.asarray(n_keys, np.int32)),
                   window, scale, out)
    return out.download(np.float32, q.shape)


def check_attn(c, q, n_keys, window, scale, H, got, what, tokens=None):
    B, T = q.shape[:2]
    G = H // c.HKV
    ts = list(range(T)) if tokens is None else tokens
    for b in range(B):
        n = max(0, min(int(n_keys[b]), c.n_table * c.page))
        for kvh in range(c.HKV):
            k, has = c.rows("k", b, kvh, n)
            v, _ = c.rows("v", b, kvh, n)
            seen = seen_by(n, T, window, has)
            for h in range(kvh * G, (kvh + 1) * G):
                want, _, tol, _ = attend(q[b, ts, h].astype(np.float64), k, v, seen[ts], scale)
                check_rows(got[b, ts, h], want, tol, (*what, b, h))


# ---- attention -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("H,HKV,HD", HEADS)
@pytest.mark.parametrize("T,page,lengths,window", [(1, 16, [1], 0), (1, 64, [0, 700, 33], 0), (1, 32, [300, 5], 100),
                                                   (5, 128, [3, 401, 5], 0), (3, 16, [90, 2, 41], 17)])
def test_attention(ctx, kv, H, HKV, HD, T, page, lengths, window):
    rng = np.random.default_rng([H, HD, T, kv, page])
    c = Pages(ctx, rng, kv, HKV, HD, page, lengths)
    q = rng.standard_normal((len(lengths), T, H, HD)).astype(np.float32)
    got = run_attn(ctx, c, q, lengths, window, 1 / np.sqrt(HD), H)
    check_attn(c, q, lengths, window, 1 / np.sqrt(HD), H, got, (kv, H, HD))
    for b, n in enumerate(lengths):
        assert np.all(got[b, :max(0, T - n)] == 0)  # tokens before the first key


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("H,HKV,HD,page,n", [(8, 2, 128, 64, 9001), (14, 2, 64, 256, 5000), (2, 1, 256, 16, 3333),
                                             (16, 1, 128, 128, 4096), (4, 1, 64, 16, 1500)])
def test_one_long_sequence(ctx, kv, H, HKV, HD, page, n):
    """Keys over many workgroups, slices that end inside pages, more pages than a wave looks up at once."""
    rng = np.random.default_rng([n, kv])
    c = Pages(ctx, rng, kv, HKV, HD, page, [n])
    for T in (1, 4):
        q = rng.standard_normal((1, T, H, HD)).astype(np.float32)
        got = run_attn(ctx, c, q, [n], 0, 0.09, H)
        check_attn(c, q, [n], 0, 0.09, H, got, (kv, T))


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("B", [63, 64, 65, 200])
def test_many_sequences(ctx, kv, B):
    """Lengths that differ a hundredfold, some of 0, and more sequences than lanes."""
    rng = np.random.default_rng([B, kv])
    lengths = [int(x) for x in np.exp(rng.uniform(0, np.log(1500), B))]
    lengths[3], lengths[B - 1], lengths[B // 2] = 0, 1700, 0
    c = Pages(ctx, rng, kv, 1, 64, 32, lengths)
    q = rng.standard_normal((B, 1, 3, 64)).astype(np.float32)
    got = run_attn(ctx, c, q, lengths, 0, 0.125, 3)
    check_attn(c, q, lengths, 0, 0.125, 3, got, (kv,))


def test_more_heads_than_counters(ctx):
    """B x KV heads past 4096: the slices are joined by a launch of their own."""
    rng = np.random.default_rng(5)
    lengths = [int(x) for x in rng.integers(0, 40, 1100)]
    lengths[700], lengths[1099] = 900, 3000
    c = Pages(ctx, rng, Q8, 4, 64, 16, lengths)
    q = rng.standard_normal((1100, 1, 8, 64)).astype(np.float32)
    got = run_attn(ctx, c, q, lengths, 0, 0.125, 8)
    some = [0, 1, 699, 700, 701, 1098, 1099]
    for b in some:
        for h in range(8):
            k, has = c.rows("k", b, h // 2, lengths[b])
            v, _ = c.rows("v", b, h // 2, lengths[b])
            want, _, tol, _ = attend(q[b, :, h].astype(np.float64), k, v, seen_by(lengths[b], 1, 0, has), 0.125)
            check_rows(got[b, :, h], want, tol, (b, h))
    assert np.all(got[[b for b in range(1100) if lengths[b] == 0]] == 0)


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("H,HKV,HD", [(14, 2, 64), (32, 8, 128), (10, 2, 128), (8, 4, 256)])
@pytest.mark.parametrize("T", [8, 16])
def test_verify_batches(ctx, kv, H, HKV, HD, T):
    """Several row tiles a KV head, the last of them not full."""
    rng = np.random.default_rng([H, T, kv])
    lengths = [1200, T, 7, 555]
    c = Pages(ctx, rng, kv, HKV, HD, 64, lengths)
    q = rng.standard_normal((4, T, H, HD)).astype(np.float32)
    for window in (0, 200, 5):
        got = run_attn(ctx, c, q, lengths, window, 0.1, H)
        check_attn(c, q, lengths, window, 0.1, H, got, (kv, T, window))


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("H,HKV,HD", [(16, 8, 64), (16, 8, 128), (8, 4, 256)])
@pytest.mark.parametrize("T,page,window", [(1, 16, 0), (1, 64, 0), (1, 32, 50), (1, 16, 300), (2, 16, 0), (3, 64, 41), (9, 16, 0),
                                           (9, 128, 33), (16, 32, 0)])
def test_many_items(ctx, kv, H, HKV, HD, T, page, window):
    """From 64 (heads of 256: 32) pairs of a sequence and a KV head on the last slice joins, and from 128 on two row tiles take
    four waves: ragged lengths, one of many slices, a page that is missing, infinities and NaN behind the last key."""
    rng = np.random.default_rng([T, HD, page, kv, window])
    lengths = [int(x) for x in rng.integers(0, 260, 24)]
    lengths[5], lengths[11], lengths[20], lengths[23] = 2900, 0, 1, 700
    c = Pages(ctx, rng, kv, HKV, HD, page, lengths)
    for b, n in enumerate(lengths):
        if n % page:
            at, slot = c.table[b, n // page], n % page
            for m in "kv":
                c.raw[m + "s" if kv == Q8 else m][at, :, slot:] = np.inf if b % 2 else np.nan
    c.table[5, 3], c.table[23, 0] = -1, c.n_pages
    c.send()
    q = rng.standard_normal((24, T, H, HD)).astype(np.float32)
    for again in range(2):  # (the counters are zero again)
        got = run_attn(ctx, c, q, lengths, window, 0.09, H)
    check_attn(c, q, lengths, window, 0.09, H, got, (kv, T, page))
    assert np.all(got[11] == 0)


@pytest.mark.parametrize("kv", [Q8, F16])
def test_counts_outside_the_pages(ctx, kv):
    """Counts in device memory are taken into the table: negative ones as 0, larger ones as all that it holds."""
    rng = np.random.default_rng(7)
    c = Pages(ctx, rng, kv, 2, 128, 16, [64, 64, 64, 64], n_table=4)
    q = rng.standard_normal((4, 2, 4, 128)).astype(np.float32)
    n = [-5, 1000, 2 ** 31 - 1, -2 ** 31]
    for window in (0, 30, 2 ** 31 - 1):
        got = run_attn(ctx, c, q, n, window, 0.1, 4)
        check_attn(c, q, [0, 64, 64, 0], min(window, 1 << 40), 0.1, 4, got, (kv, window))
        assert np.all(got[[0, 3]] == 0)


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("HD", [64, 128])
def test_missing_and_shared_pages(ctx, kv, HD):
    """Entries that are no page (their keys are nobody's) and pages that several sequences share."""
    rng = np.random.default_rng([9, HD])
    lengths = [300, 290, 40, 200]
    c = Pages(ctx, rng, kv, 2, HD, 16, lengths)
    c.table[0, 3], c.table[0, 7], c.table[0, 8] = -1, c.n_pages, 2 ** 31 - 1
    c.table[1, :10] = c.table[3, :10]
    c.table[2, :3] = -7
    c.send()
    q = rng.standard_normal((4, 3, 4, HD)).astype(np.float32)
    for window in (0, 100):
        got = run_attn(ctx, c, q, lengths, window, 0.1, 4)
        check_attn(c, q, lengths, window, 0.1, 4, got, (kv, HD, window))
        assert np.all(got[2] == 0)


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("H,HKV,HD", [(14, 2, 64), (8, 2, 128), (8, 4, 256)])
def test_nonfinite_rows_that_are_not_read(ctx, kv, H, HKV, HD):
    """NaN and infinities behind the sequence, in other pages, in keys of later tokens and in front of the window
    do not reach a token; those of keys that it reads do."""
    rng = np.random.default_rng([11, HD, kv])
    n, T, page = 141, 6, 32
    c = Pages(ctx, rng, kv, HKV, HD, page, [n, 60])

    def put(pos, x):
        p, s = c.table[0, pos // page], pos % page
        for m in "kv":
            c.raw[m + "s" if kv == Q8 else m][p, :, s] = x

    spare = [p for p in range(c.n_pages) if p not in c.table]
    for m in "kv":
        c.raw[m + "s" if kv == Q8 else m][spare] = np.nan
    put(n - 2, np.nan)  # token 4 is the first that reads it
    put(n - 1, np.inf)
    for pos in range(n, -(-n // page) * page):
        put(pos, np.nan)
    c.send()
    q = rng.standard_normal((2, T, H, HD)).astype(np.float32)
    got = run_attn(ctx, c, q, [n, 60], 0, 0.1, H)
    check_attn(c, q[:1], [n], 0, 0.1, H, got, (kv,), tokens=[0, 1, 2, 3])
    assert np.all(np.isnan(got[0, 4:]))
    assert np.all(np.isfinite(got[1]))
    # In front of the window: tokens 2.. read keys from n - 6 + 3 - 80 on.
    c2 = Pages(ctx, np.random.default_rng(12), kv, HKV, HD, page, [n])
    first = n - T + 1 - 80 + 2  # the first key of token 2
    p, s = c2.table[0, (first - 1) // page], (first - 1) % page
    c2.raw["vs" if kv == Q8 else "v"][p, :, s] = np.inf
    c2.send()
    got = run_attn(ctx, c2, q[:1], [n], 80, 0.1, H)
    check_attn(c2, q[:1], [n], 80, 0.1, H, got, (kv,), tokens=[2, 3, 4, 5])
    assert not np.any(np.isfinite(got[0, :2]))


def test_scores_of_minus_infinity(ctx):
    """Rows whose scores are all minus infinity count as rows without a key; one finite score takes all the weight."""
    rng = np.random.default_rng(13)
    c = Pages(ctx, rng, F16, 1, 64, 16, [20])
    for i in range(2):
        c.raw["k"][c.table[0, i]] = np.float16(-60000)
    c.send()
    q = np.full((1, 1, 2, 64), 3e38, np.float32)
    q[0, 0, 1] = rng.standard_normal(64)
    got = run_attn(ctx, c, q, [20], 0, 1.0, 2)
    assert np.all(got[0, 0, 0] == 0) and np.all(np.isfinite(got[0, 0, 1]))


@pytest.mark.parametrize("kv", [Q8, F16])
def test_large_scores(ctx, kv):
    rng = np.random.default_rng(14)
    c = Pages(ctx, rng, kv, 2, 128, 64, [500], std=8.0)
    q = (rng.standard_normal((1, 1, 8, 128)) * 40).astype(np.float32)
    got = run_attn(ctx, c, q, [500], 0, 1.0, 8)
    check_attn(c, q, [500], 0, 1.0, 8, got, (kv,))


def test_calls_in_turn(ctx):
    """Calls of different sizes one after another without a wait, each twice with the same bits: the scratch and the
    counters are as the next call needs them."""
    rng = np.random.default_rng(15)
    jobs = []
    for kv, HKV, H, HD, page, lengths, T in ((Q8, 8, 32, 128, 64, [2000, 17, 900], 1), (F16, 2, 14, 64, 16, [60], 1),
                                             (Q8, 2, 14, 64, 16, [700, 0], 9), (F16, 1, 8, 256, 256, [3000], 2)):
        c = Pages(ctx, rng, kv, HKV, HD, page, lengths)
        q = rng.standard_normal((len(lengths), T, H, HD)).astype(np.float32)
        jobs.append((c, q, lengths, H, ctx.to_device(q), ctx.to_device(np.array(lengths, np.int32)),
                     [ctx.alloc(q.nbytes) for _ in range(3)]))
    for turn in range(3):
        for c, q, lengths, H, qd, nd, outs in jobs:
            ctx.attn_paged(qd, *q.shape[:2], H, c.HKV, c.HD, *c.args, c.n_table, nd, 0, 0.1, outs[turn])
    for c, q, lengths, H, qd, nd, outs in jobs:
        got = [o.download(np.float32, q.shape) for o in outs]
        check_attn(c, q, lengths, 0, 0.1, H, got[0], (H,))
        assert all(np.array_equal(got[0].view(np.uint32), g.view(np.uint32)) for g in got[1:])


def test_two_contexts_at_once(ctx):
    """Calls of two contexts (streams, scratch and counters of their own) in flight together: the bits of calls alone."""
    other = ts5hip.Context(0)
    try:
        jobs = []
        for x, seed in ((ctx, 1), (other, 2)):
            rng = np.random.default_rng(seed)
            for kv, T, lengths in ((Q8, 1, [3000, 900, 5, 260] * 3), (F16, 1, [8000]), (Q8, 6, [1500, 40])):
                c = Pages(x, rng, kv, 8, 128, 32, lengths)
                q = rng.standard_normal((len(lengths), T, 32, 128)).astype(np.float32)
                args = x.to_device(q), x.to_device(np.array(lengths, np.int32)), [x.alloc(q.nbytes) for _ in range(9)]
                alone = run_attn(x, c, q, lengths, 0, 0.09, 32)
                jobs.append((x, c, q, alone, *args))
        ctx.sync(), other.sync()
        for turn in range(9):
            for x, c, q, alone, qd, nd, outs in jobs[turn % 3::3]:
                x.attn_paged(qd, *q.shape[:2], 32, 8, 128, *c.args, c.n_table, nd, 0, 0.09, outs[turn])
            for x, c, q, alone, qd, nd, outs in jobs:
                x.attn_paged(qd, *q.shape[:2], 32, 8, 128, *c.args, c.n_table, nd, 0, 0.09, outs[turn])
        for x, c, q, alone, qd, nd, outs in jobs:
            for out in outs:
                assert np.array_equal(out.download(np.float32, q.shape).view(np.uint32), alone.view(np.uint32))
        del jobs, x, c, q, alone, qd, nd, outs, out, args  # (the other context's buffers, before it)
    finally:
        other.close()


def test_same_as_a_contiguous_cache(ctx):
    """Sequences of one length in pages and in caches of their own: the same attention."""
    rng = np.random.default_rng(16)
    n, H, HKV, HD = 1000, 32, 8, 128
    c = Pages(ctx, rng, Q8, HKV, HD, 64, [n, n])
    slots = c.n_table * 64
    whole = {}
    for m in c.raw:
        x = np.zeros((2, HKV, slots, *c.raw[m].shape[3:]), c.raw[m].dtype)
        for b in range(2):
            for i in range(-(-n // 64)):
                x[b, :, i * 64:(i + 1) * 64] = c.raw[m][c.table[b, i]]
        whole[m] = ctx.to_device(x)
    q = rng.standard_normal((2, 1, H, HD)).astype(np.float32)
    got = run_attn(ctx, c, q, [n, n], 0, 0.088, H)
    out = ctx.alloc(q.nbytes)
    ctx.attn_decode(ctx.to_device(q), 2, H, HKV, HD, whole["k"], whole["ks"], whole["v"], whole["vs"], slots,
                    ctx.to_device(np.full(2, n, np.int32)), 1, 0.088, out)
    want = out.download(np.float32, q.shape)
    assert np.linalg.norm(got - want) <= 2e-6 * np.linalg.norm(want)


# ---- rows into the pages -----------------------------------------------------------------------------------

def rope_angles(n_pos, n_rot, base=10000.0):
    a = np.arange(n_pos)[:, None] * base ** (-np.arange(0, n_rot, 2) / max(n_rot, 1))
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def rotated(x, cs, n_rot, neox):
    """x [token][head][HD] (float64), cs [token][n_rot / 2][2]."""
    y, half = x.copy(), n_rot // 2
    a, b = (np.arange(half), np.arange(half) + half) if neox else (2 * np.arange(half), 2 * np.arange(half) + 1)
    c, s = cs[:, None, :, 0].astype(np.float64), cs[:, None, :, 1].astype(np.float64)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def append(ctx, c, qkv, seq, pos, H, n_rot, neox, cs, q_out=None, **more):
    ntok = len(seq)
    q_out = q_out or ctx.to_device(np.full((ntok, H * c.HD), 7.0, np.float32))
    up = {n: ctx.to_device(a) for n, a in more.items() if a is not None}
    ctx.rope_kv_append_paged(ctx.to_device(qkv), ntok, ctx.to_device(np.asarray(seq, np.int32)),
                             ctx.to_device(np.asarray(pos, np.int32)), H, c.HKV, c.HD, n_rot, neox, ctx.to_device(cs), len(cs),
                             q_out, *c.args, *c.table.shape, eps=1e-5, **up)
    return q_out.download(np.float32, (ntok, H, c.HD))


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("H,HKV,HD", [(14, 2, 64), (32, 8, 128), (5, 1, 128), (8, 4, 256), (2, 2, 64)])
@pytest.mark.parametrize("n_rot,neox,bias,norms", [("all", 0, False, False), ("all", 1, True, False), ("all", 1, False, True),
                                                   (32, 0, True, True), (22, 1, False, True), (10, 1, True, False), (0, 0, False, False),
                                                   (6, 0, False, False)])
def test_append(ctx, kv, H, HKV, HD, n_rot, neox, bias, norms):
    """Values as their roundings allow: fp32 sums of a bias, a norm and a rotation are off by at most 8 half steps of the
    largest value in the head (the bias, three products and the sum of the rotation; the norm's factor), the norm's sum
    of HD squares by as many half steps of itself; a cached value by half a step of its scale (or of f16) more."""
    rng = np.random.default_rng([H, HD, n_rot if n_rot != "all" else 1, neox, kv])
    n_rot = HD if n_rot == "all" else n_rot
    lengths = [70, 40, 3]
    c = Pages(ctx, rng, kv, HKV, HD, 16, lengths)
    before = {n: a.copy() for n, a in c.raw.items()}
    seq = [0, 0, 1, -1, 2, 0, 3, 1, 0, 2, 1]
    pos = [69, 5, 39, 0, 2, 0, 0, 48, -1, 70, 17]  # (the 4th and the 7th: no sequence; 48 and 70: no page or no row; -1)
    ok = [i for i in range(len(seq)) if 0 <= seq[i] < 3 and 0 <= pos[i] < 70 and c.table[seq[i], pos[i] // 16] >= 0]
    assert len(ok) == 6
    cs = rope_angles(70, n_rot) if n_rot else np.zeros((70, 0, 2), np.float32)
    cs_dev = cs if n_rot else np.zeros((70, 2), np.float32)
    width = (H + 2 * HKV) * HD
    qkv = rng.standard_normal((len(seq), width)).astype(np.float32)
    more = dict(bias=rng.standard_normal(width).astype(np.float32) if bias else None,
                q_norm=(1 + 0.3 * rng.standard_normal(HD)).astype(np.float32) if norms else None,
                k_norm=(1 + 0.3 * rng.standard_normal(HD)).astype(np.float32) if norms else None)
    got_q = append(ctx, c, qkv, seq, pos, H, n_rot, neox, cs_dev, **more)
    after = c.fetch()
    x = qkv.astype(np.float64) + (more["bias"].astype(np.float64) if bias else 0)
    x = x.reshape(len(seq), -1, HD)
    parts = {"q": x[:, :H], "k": x[:, H:H + HKV], "v": x[:, H + HKV:]}
    for n in "qk":
        y = parts[n]
        if norms:
            y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + 1e-5) * more[n + "_norm"].astype(np.float64)
        parts[n] = rotated(y, cs[np.clip(pos, 0, 69)], n_rot, neox)
    half = 2.0 ** -24
    steps = (8 + (HD if norms else 0)) * half

    def tol(y):
        return steps * (np.abs(y).max(-1, keepdims=True) * 2 + (np.abs(x).max() if bias else 0))

    err = np.abs(got_q[ok] - parts["q"][ok])
    assert np.all(err <= tol(parts["q"][ok])), (err / tol(parts["q"][ok])).max()
    left = [i for i in range(len(seq)) if i not in ok]
    assert np.all(got_q[left] == 7.0)
    touched = np.zeros((c.n_pages, 16), bool)
    for i in ok:
        p, s = c.table[seq[i], pos[i] // 16], pos[i] % 16
        touched[p, s] = True
        for n in "kv":
            want, got = parts[n][i], c.values(n, after)[p, :, s]
            t = tol(want)
            if kv == F16:
                step = np.maximum(np.abs(want) * 2.0 ** -11, 2.0 ** -25)
            else:  # half a scale; a value at the largest is cut by the scale's own rounding (127 * 2^-11 of a step)
                g = np.abs(want).reshape(HKV, -1, 32).max(-1)
                step = np.repeat(g / 127 * (1 + 2.0 ** -11) * (0.5 + 127 * 2.0 ** -11), 32, axis=-1)
            assert np.all(np.abs(got - want) <= step * (1 + 1e-6) + 2 * t), (n, i)
    for n, a in after.items():  # nothing else is written
        keep = ~touched[:, None, :].repeat(HKV, 1)
        assert np.array_equal(a[keep], before[n][keep]), n


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("H,HKV,HD,neox,bias", [(32, 8, 128, 0, False), (14, 2, 64, 1, True), (8, 4, 256, 1, False)])
def test_append_as_into_a_contiguous_cache(ctx, kv, H, HKV, HD, neox, bias):
    """The same bits as ts5hip_rope_kv_append_at writes, and the same rows of q."""
    rng = np.random.default_rng([21, HD, kv])
    n, first = 150, 37
    c = Pages(ctx, rng, kv, HKV, HD, 32, [first + n])
    width = (H + 2 * HKV) * HD
    qkv = rng.standard_normal((n, width)).astype(np.float32) * 3
    b = rng.standard_normal(width).astype(np.float32) if bias else None
    cs = rope_angles(first + n, HD)
    pos = np.arange(first, first + n, dtype=np.int32)
    got_q = append(ctx, c, qkv, np.zeros(n), pos, H, HD, neox, cs, bias=b)
    after = c.fetch()
    slots = 256
    flat = {m: ctx.to_device(np.zeros((HKV, slots, *a.shape[3:]), a.dtype)) for m, a in c.raw.items()}
    q_out = ctx.alloc(n * H * HD * 4)
    ctx.rope_kv_append_at(ctx.to_device(qkv), n, ctx.to_device(pos), ctx.to_device(np.array([first], np.int32)), H, HKV, HD, HD,
                          neox, ctx.to_device(cs), len(cs), slots, kv, q_out, flat["k"], flat.get("ks"), flat["v"],
                          flat.get("vs"), bias=ctx.to_device(b) if bias else None, eps=1e-5)
    assert np.array_equal(q_out.download(np.float32, got_q.shape).view(np.uint32), got_q.view(np.uint32))
    for m, a in after.items():
        want = flat[m].download(a.dtype, (HKV, slots, *a.shape[3:]))
        for p in pos:
            assert np.array_equal(a[c.table[0, p // 32], :, p % 32], want[:, p]), (m, p)


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("H,HKV,HD,n,n_rot,neox,bias,norms", [
    (32, 8, 128, 2221, 128, 0, False, False), (40, 8, 128, 1903, 128, 1, True, False), (14, 2, 64, 6659, 64, 1, True, False),
    (14, 2, 64, 6658, 22, 0, False, True), (8, 4, 256, 3331, 256, 1, False, True), (8, 4, 256, 3329, 0, 0, True, False)])
def test_append_of_many_tokens(ctx, kv, H, HKV, HD, n, n_rot, neox, bias, norms):
    """From 13312 workgroups of rows on (6, 7, 2 and 4 of them a token here) a thread takes four tokens: the same bits as in
    calls of 100 tokens, whatever the count, tokens without a place among them."""
    rng = np.random.default_rng([31, HD, n, kv])
    lengths = [n // 2, n - n // 2]
    c = Pages(ctx, rng, kv, HKV, HD, 64, lengths)
    seq = np.repeat([0, 1], lengths).astype(np.int32)
    pos = np.concatenate([np.arange(m) for m in lengths]).astype(np.int32)
    order = rng.permutation(n)
    seq, pos = seq[order], pos[order]
    seq[rng.integers(0, n, 40)] = -1
    pos[rng.integers(0, n, 40)] = -5
    width = (H + 2 * HKV) * HD
    qkv = rng.standard_normal((n, width)).astype(np.float32) * 3
    cs = rope_angles(max(lengths), n_rot) if n_rot else np.zeros((max(lengths), 2), np.float32)
    more = dict(bias=rng.standard_normal(width).astype(np.float32) if bias else None,
                q_norm=(1 + 0.3 * rng.standard_normal(HD)).astype(np.float32) if norms else None,
                k_norm=(1 + 0.3 * rng.standard_normal(HD)).astype(np.float32) if norms else None)
    parts = [append(ctx, c, qkv[i:i + 100], seq[i:i + 100], pos[i:i + 100], H, n_rot, neox, cs, **more) for i in range(0, n, 100)]
    want = c.fetch()
    for name, b in c.dev.items():
        b.upload(c.raw[name])
    got_q = append(ctx, c, qkv, seq, pos, H, n_rot, neox, cs, **more)
    assert np.array_equal(got_q.view(np.uint32), np.concatenate(parts).view(np.uint32))
    for name, a in c.fetch().items():
        assert np.array_equal(a.view(np.uint8), want[name].view(np.uint8)), name


# ---- rows back ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("HKV,HD", [(1, 64), (2, 64), (8, 128), (4, 256), (3, 128)])
@pytest.mark.parametrize("out", [ts5hip.F32, ts5hip.F16])
def test_read(ctx, kv, HKV, HD, out):
    """Every value as it stands for, exactly (f32) or to the nearest half; rows of tokens without a place stay."""
    rng = np.random.default_rng([31, HD, HKV, kv])
    c = Pages(ctx, rng, kv, HKV, HD, 32, [75, 130])
    c.table[1, 2] = -1
    c.send()
    seq = np.concatenate([np.zeros(75), np.ones(130), [-1, 2, 0, 1, 0, 0]]).astype(np.int32)
    pos = np.concatenate([np.arange(75), np.arange(130)[::-1], [3, 3, -1, 2 ** 31 - 1, 10 ** 6, 74]]).astype(np.int32)
    dtype = np.float32 if out == ts5hip.F32 else np.float16
    outs = [ctx.to_device(np.full((len(seq), HKV * HD), 5, dtype)) for _ in range(2)]
    ctx.kv_read_paged(len(seq), ctx.to_device(seq), ctx.to_device(pos), HKV, HD, *c.args, *c.table.shape, out, *outs)
    for n, o in zip("kv", outs):
        got, x = o.download(dtype, (len(seq), HKV, HD)), c.values(n)
        for i, (s, p) in enumerate(zip(seq, pos)):
            page = c.table[s, p // 32] if 0 <= s < 2 and 0 <= p < c.n_table * 32 else -1
            want = np.full((HKV, HD), 5, dtype) if page < 0 else x[page, :, p % 32].astype(dtype)
            assert np.array_equal(got[i], want), (n, i)


@pytest.mark.parametrize("n", [1, 3, 4, 5])
def test_read_few(ctx, n):
    rng = np.random.default_rng(n)
    c = Pages(ctx, rng, Q8, 2, 128, 16, [40])
    outs = [ctx.to_device(np.full((8, 256), 5, np.float32)) for _ in range(2)]
    pos = np.array([39, 0, 16, 15, 7][:n], np.int32)
    ctx.kv_read_paged(n, ctx.to_device(np.zeros(n, np.int32)), ctx.to_device(pos), 2, 128, *c.args, *c.table.shape, ts5hip.F32, *outs)
    for m, o in zip("kv", outs):
        got = o.download(np.float32, (8, 2, 128))
        assert np.array_equal(got[:n], c.values(m)[c.table[0, pos // 16], :, pos % 16].astype(np.float32))
        assert np.all(got[n:] == 5)


def test_pools_past_4_gib(ctx):
    """Pages whose byte offsets pass 32 bits: written, attended to and read back."""
    HKV, HD, page, H, n_pages = 8, 256, 256, 8, 4400  # 1 MiB of K a page (f16)
    k, v = ctx.alloc(n_pages << 20), ctx.alloc(n_pages << 20)
    table = np.array([[n_pages - 1, 4097, 0, -1], [2049, -1, -1, -1]], np.int32)
    args = (F16, k, None, v, None, n_pages, page, ctx.to_device(table))
    rng = np.random.default_rng(41)
    lengths = [600, 130]
    seq = np.concatenate([np.full(n, b) for b, n in enumerate(lengths)]).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in lengths]).astype(np.int32)
    qkv = rng.standard_normal((len(seq), (H + 2 * HKV) * HD)).astype(np.float32)
    q_out = ctx.alloc(len(seq) * H * HD * 4)
    ctx.rope_kv_append_paged(ctx.to_device(qkv), len(seq), ctx.to_device(seq), ctx.to_device(pos), H, HKV, HD, 0, 0,
                             ctx.to_device(np.zeros((600, 2), np.float32)), 600, q_out, *args, 2, 4)
    x = qkv.reshape(len(seq), H + 2 * HKV, HD)
    half = x[:, H:].astype(np.float16)
    outs = [ctx.alloc(len(seq) * HKV * HD * 2) for _ in range(2)]
    ctx.kv_read_paged(len(seq), ctx.to_device(seq), ctx.to_device(pos), HKV, HD, *args, 2, 4, ts5hip.F16, *outs)
    for i, o in enumerate(outs):
        assert np.array_equal(o.download(np.float16, (len(seq), HKV, HD)), half[:, i * HKV:(i + 1) * HKV])
    q = rng.standard_normal((2, 2, H, HD)).astype(np.float32)
    out = ctx.alloc(q.nbytes)
    ctx.attn_paged(ctx.to_device(q), 2, 2, H, HKV, HD, *args, 4, ctx.to_device(np.array(lengths, np.int32)), 0, 0.06, out)
    got = out.download(np.float32, q.shape)
    for b, n in enumerate(lengths):
        rows = half[seq == b].astype(np.float64)
        for h in range(H):
            want, _, tol, _ = attend(q[b, :, h].astype(np.float64), rows[:, h], rows[:, HKV + h],
                                     seen_by(n, 2, 0, np.ones(n, bool)), 0.06)
            check_rows(got[b, :, h], want, tol, (b, h))


@pytest.mark.parametrize("kv", [Q8, F16])
@pytest.mark.parametrize("HKV,HD,n", [(8, 128, 7), (2, 64, 7), (4, 256, 7), (8, 128, 3400)])
def test_append_of_values_that_are_not_finite(ctx, kv, HKV, HD, n):
    """NaN and infinities in a token's K and V come back as such, an infinity with its sign: f16 caches round each value by
    itself; of a q8 cache's 32 values that share a scale none is finite then. All others have the bits that they have
    without them. (3400 tokens of 6 workgroups of rows: four tokens a thread.)"""
    rng = np.random.default_rng([61, HD, n, kv])
    H = 2 * HKV if n < 100 else 32
    c = Pages(ctx, rng, kv, HKV, HD, 16, [n])
    seq, pos = np.zeros(n, np.int32), np.arange(n, dtype=np.int32)
    cs = np.zeros((n, 2), np.float32)
    good = rng.standard_normal((n, H + 2 * HKV, HD)).astype(np.float32)
    bad = good.copy()
    hurt = np.zeros((n, 2 * HKV, HD // 32), bool)  # groups of 32 with such a value
    for t in range(n):
        for _ in range(4):
            head, d = rng.integers(0, 2 * HKV), rng.integers(0, HD)
            bad[t, H + head, d] = rng.choice(np.array([np.nan, -np.nan, np.inf, -np.inf], np.float32))
            hurt[t, head, d // 32] = True
    bad[0, H, :32], hurt[0, 0, 0] = np.nan, True  # all of a group
    caches = []
    for x in (good, bad):
        for name, b in c.dev.items():
            b.upload(c.raw[name])
        append(ctx, c, x.reshape(n, -1), seq, pos, H, 0, 0, cs)
        caches.append(c.fetch())
    page, slot = c.table[0, pos // 16], pos % 16
    for i, name in enumerate("kv"):
        want = bad[:, H + i * HKV:H + (i + 1) * HKV]
        groups = hurt[:, i * HKV:(i + 1) * HKV]
        was, got = (c.values(name, raw)[page, :, slot] for raw in caches)
        in_group = np.repeat(groups, 32, axis=-1)
        assert np.array_equal(got[~in_group], was[~in_group])
        if kv == F16:
            assert np.array_equal(got[in_group], want[in_group].astype(np.float16).astype(np.float64), equal_nan=True)
            continue
        assert not np.any(np.isfinite(got[in_group]))
        has_nan = np.repeat(np.isnan(want).reshape(n, HKV, -1, 32).any(-1), 32, axis=-1)
        assert np.all(np.isnan(got[has_nan]))
        signed = np.isinf(want) & ~has_nan
        assert signed.any() and np.array_equal(got[signed], want[signed].astype(np.float64))
    # Read back they are the same.
    outs = [ctx.alloc(n * HKV * HD * 4) for _ in range(2)]
    ctx.kv_read_paged(n, ctx.to_device(seq), ctx.to_device(pos), HKV, HD, *c.args, *c.table.shape, ts5hip.F32, *outs)
    for name, o in zip("kv", outs):
        assert np.array_equal(o.download(np.float32, (n, HKV, HD)), c.values(name, caches[1])[page, :, slot].astype(np.float32),
                              equal_nan=True)


def test_joins_of_2_32_values():
    """4096 sequences of 16 tokens of 256 heads of 256, 16 GiB of rows: more threads than one dimension of a grid takes join
    the slices. Most sequences have no key; the first, one in the middle and the last have keys in several slices."""
    ctx = ts5hip.Context(0)
    try:
        rng = np.random.default_rng(71)
        B, T, H, HKV, HD, n_table = 4096, 16, 256, 16, 256, 64
        k, v = (rng.standard_normal((n_table, HKV, 16, HD)).astype(np.float16) for _ in range(2))
        kd, vd = ctx.to_device(k), ctx.to_device(v)
        table = ctx.to_device(np.tile(np.arange(n_table, dtype=np.int32), (B, 1)))
        lengths = np.zeros(B, np.int32)
        lengths[[0, 2047, B - 1]] = 900, 1024, 700
        row = T * H * HD * 4  # bytes of a sequence
        q, out = ctx.alloc(B * row), ctx.alloc(B * row)
        rows = {b: rng.standard_normal((T, H, HD)).astype(np.float32) for b in (0, 2047, B - 1)}
        for b, x in rows.items():
            ctx.check(ts5hip.lib().ts5hip_upload(ctx.h, q.ptr + b * row, x.ctypes.data, x.nbytes))
        ctx.attn_paged(q, B, T, H, HKV, HD, F16, kd, None, vd, None, n_table, 16, table, n_table, ctx.to_device(lengths), 0, 0.06,
                       out)
        kk, vv = (x.astype(np.float64).transpose(1, 0, 2, 3).reshape(HKV, -1, HD) for x in (k, v))
        for b, x in rows.items():
            got, n = out.download(np.float32, (T, H, HD), b * row), int(lengths[b])
            seen = seen_by(n, T, 0, np.ones(n, bool))
            for h in (0, 15, 100, 255):
                want, _, tol, _ = attend(x[:, h].astype(np.float64), kk[h // 16, :n], vv[h // 16, :n], seen, 0.06)
                check_rows(got[:, h], want, tol, (b, h))
        for b in (1, 2046, 2048, B - 2):
            assert np.all(out.download(np.float32, (T * H * HD,), b * row) == 0)
        del q, out, kd, vd, table
    finally:
        ctx.close()
