"""Drafted tokens judged by the target's and the draft's probabilities, through the C ABI, against float64 numpy: kept
drafts and drawn tokens are equal (both sides compute in 64 bits, so that two orders of a sum differ by about 1e-15, and
a bound within that of a cumulative weight is not met by chance), log-probabilities to their rounding to fp32."""
import numpy as np
import pytest

from test_gpu_paged import F16, Q8, Pages, append, rope_angles
from tokenstation5_amd import ts5hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ts5hip.Context(0)
    yield c
    c.close()


def probabilities(row, t):
    """(softmax of row / t, log of it), or None where there is no distribution."""
    x = row.astype(np.float64)
    if np.isnan(x).any() or x.max() == np.inf or x.max() == -np.inf:
        return None
    with np.errstate(invalid="ignore"):
        z = (x - x.max()) / t
    z[x == -np.inf] = -np.inf
    w = np.exp(z)
    with np.errstate(divide="ignore"):
        return w / w.sum(), z - np.log(w.sum())


def judge(logits, draft_logits, drafts, t, u):
    """One sequence: (tokens, log-probabilities). logits [n + 1][V], drafts [n], u [n + 1 of n_draft's, the last the draw's]."""
    tokens, logps = [], []
    for i in range(len(drafts) + 1):
        got = probabilities(logits[i], t if t > 0 else 1.0)
        if got is None:
            return tokens, logps
        p, lp = got
        if not t > 0:
            best = int(np.argmax(logits[i]))
            if i < len(drafts) and drafts[i] == best:
                tokens.append(best), logps.append(0.0)
                continue
            return tokens + [best], logps + [0.0]
        w = p
        if i < len(drafts):
            d, q = int(drafts[i]), None
            inside = 0 <= d < len(p)
            if draft_logits is None:
                q = np.zeros_like(p)
                if inside:
                    q[d] = 1.0
            else:
                got = probabilities(draft_logits[i], t)
                q = got[0] if got else None
            if inside and q is not None and u[i] * q[d] < p[d]:
                tokens.append(d), logps.append(lp[d])
                continue
            if q is not None:
                w = np.maximum(p - q, 0.0)
                if not w.sum() > 0:
                    w = p
        c = np.cumsum(w)
        at = int(np.searchsorted(c, np.float64(u[-1]) * c[-1], side="right"))
        at = min(at, int(np.nonzero(w)[0][-1]))
        return tokens + [at], logps + [lp[at]]


def run(ctx, logits, draft_logits, drafts, n_draft, temp, uni, V=None, outs=None):
    B, T1, ld = logits.shape
    T = T1 - 1
    tokens, n, logp = outs or (ctx.to_device(np.full((B, T1), 99, np.int32)), ctx.to_device(np.full(B, 99, np.int32)),
                               ctx.to_device(np.full((B, T1), 99, np.float32)))
    ctx.verify_drafts(ctx.to_device(logits), ld, None if draft_logits is None else ctx.to_device(draft_logits),
                      0 if draft_logits is None else draft_logits.shape[2], V or ld, B, T,
                      ctx.to_device(drafts.astype(np.int32)) if T else None,
                      None if n_draft is None else ctx.to_device(np.asarray(n_draft, np.int32)),
                      ctx.to_device(np.asarray(temp, np.float32)), ctx.to_device(uni.astype(np.float32)), tokens, n, logp)
    return tokens.download(np.int32, (B, T1)), n.download(np.int32, (B,)), logp.download(np.float32, (B, T1))


def check(logits, draft_logits, drafts, n_draft, temp, uni, got, V=None, what=()):
    V = V or logits.shape[2]
    T = logits.shape[1] - 1
    tokens, counts, logp = got
    for b in range(len(logits)):
        n = T if n_draft is None else max(0, min(int(n_draft[b]), T))
        u = np.append(uni[b, :n], uni[b, T])
        want, lps = judge(logits[b, :n + 1, :V], None if draft_logits is None else draft_logits[b, :n, :V], drafts[b, :n],
                          float(np.float32(temp[b])), u)
        assert counts[b] == len(want) and list(tokens[b]) == want + [-1] * (T + 1 - len(want)), (*what, b, want, tokens[b])
        lps = np.array(lps + [0.0] * (T + 1 - len(want)))
        assert np.all(np.abs(logp[b] - lps) <= np.abs(lps) * 2.0 ** -23 + 1e-12), (*what, b)


def inputs(rng, B, T, V, model, ld=None, noise=0.8):
    ld = ld or V
    logits = (2 * rng.standard_normal((B, T + 1, ld))).astype(np.float32)
    for _ in range(3):
        np.put_along_axis(logits, rng.integers(0, V, (B, T + 1, 1)), rng.uniform(5, 9, (B, T + 1, 1)).astype(np.float32), 2)
    temp = rng.uniform(0.5, 1.3, B).astype(np.float32)
    draft = (logits[:, :T] + noise * rng.standard_normal((B, T, ld))).astype(np.float32) if model else None
    rows = (draft if model else logits[:, :T])[:, :, :V] / temp[:, None, None]
    drafts = (rows + rng.gumbel(size=rows.shape)).argmax(-1) if T else np.zeros((B, 0), np.int64)
    return logits, draft, drafts, temp, rng.random((B, T + 1), dtype=np.float32)


@pytest.mark.parametrize("model", [False, True])
@pytest.mark.parametrize("B,T,V,ld", [(1, 0, 1000, 1000), (3, 1, 4096, 4096), (5, 4, 4097, 4100), (2, 5, 50257, 50257),
                                      (4, 7, 8191, 8193), (40, 3, 333, 333), (2, 63, 700, 701), (300, 2, 37, 37), (1, 5, 151936, 151936)])
def test_verify(ctx, model, B, T, V, ld):
    rng = np.random.default_rng([B, T, V, model])
    logits, draft, drafts, temp, uni = inputs(rng, B, T, V, model, ld)
    if ld > V:  # what is behind a row's entries does not count
        logits[:, :, V:] = np.nan
        if model:
            draft[:, :, V:] = np.inf
    check(logits, draft, drafts, None, temp, uni, run(ctx, logits, draft, drafts, None, temp, uni, V), V)
    n = rng.integers(-1, T + 3, B)
    check(logits, draft, drafts, n, temp, uni, run(ctx, logits, draft, drafts, n, temp, uni, V), V)


@pytest.mark.parametrize("model", [False, True])
def test_the_best_token(ctx, model):
    """Temperature 0, below 0 or NaN: the first of the largest entries, whatever the draft's probabilities."""
    rng = np.random.default_rng(3)
    logits, draft, drafts, temp, uni = inputs(rng, 12, 4, 9001, model)
    drafts = logits[:, :4].argmax(-1)
    logits[1, 2, [4, 8000]] = 50.0  # equal: the first
    drafts[1, 2] = 8000
    logits[2, 1, [17, 6000]] = 50.0
    drafts[2, 1] = 17
    drafts[3, 0], drafts[4, 3], drafts[5, 2] = 5, -1, 9001
    temp[:6] = [0.0, 0.0, -1.0, np.nan, 0.0, -0.0]
    got = run(ctx, logits, draft, drafts, None, temp, uni)
    check(logits, draft, drafts, None, temp, uni, got)
    assert got[1][0] == 5 and list(got[0][1][:3]) == [*drafts[1, :2], 4] and got[1][1] == 3 and got[1][2] == 5


@pytest.mark.parametrize("model", [False, True])
def test_masked_entries(ctx, model):
    """Entries of minus infinity have no probability; whole slices of them; one entry alone."""
    rng = np.random.default_rng(4)
    B, T, V = 8, 3, 13000
    logits, draft, drafts, temp, uni = inputs(rng, B, T, V, model)
    logits[0, :, 4096:8192] = -np.inf
    logits[1, :, :12999] = -np.inf
    logits[2, :, 1:] = -np.inf
    logits[3, 0] = np.where(rng.random(V) < 0.9, -np.inf, logits[3, 0])
    if model:
        draft[4, 0, :12000] = -np.inf
        draft[5, 0] = np.where(np.arange(V) == drafts[5, 0], 0.0, -np.inf)  # certain
    drafts[6, 1], drafts[7, 0] = V, -1
    for trial in range(6):
        uni = rng.random((B, T + 1), dtype=np.float32)
        if trial == 0:
            uni[:] = 0
        if trial == 1:
            uni[:] = 1 - 2.0 ** -24
        check(logits, draft, drafts, None, temp, uni, run(ctx, logits, draft, drafts, None, temp, uni), what=(trial,))


@pytest.mark.parametrize("model", [False, True])
def test_rows_without_a_distribution(ctx, model):
    """NaN, plus infinity or only minus infinity: a sequence ends at such a row of the target's, and does not keep a draft
    of such a row of the draft's."""
    rng = np.random.default_rng(5)
    B, T, V = 9, 3, 5000
    logits, draft, drafts, temp, uni = inputs(rng, B, T, V, model, noise=0.0)
    uni[:, :T] = 0  # everything that can be kept is
    logits[0, 1, 4500], logits[1, 0, 3], logits[2, 3] = np.nan, np.inf, -np.inf
    logits[3, 1], temp[3] = np.nan, 0.0
    drafts[3] = [logits[3, 0].argmax(), 1, 2]
    if model:
        draft[4, 1, 17], draft[5, 0, 4999], draft[6, 2] = np.nan, np.inf, -np.inf
    got = run(ctx, logits, draft, drafts, None, temp, uni)
    check(logits, draft, drafts, None, temp, uni, got)
    assert list(got[1][:4]) == [1, 0, 3, 1]
    if model:
        assert list(got[1][4:7]) == [2, 1, 3]


def test_equal_rows(ctx):
    """A draft model that is the target: every draft is kept. Entries all alike: cumulative weights that bounds meet
    exactly, on whole numbers."""
    rng = np.random.default_rng(6)
    logits, draft, drafts, temp, uni = inputs(rng, 6, 5, 20000, True, noise=0.0)
    uni[:, :5] = 1 - 2.0 ** -24
    got = run(ctx, logits, draft, drafts, None, temp, uni)
    check(logits, draft, drafts, None, temp, uni, got)
    assert np.all(got[1] == 6)
    B, V = 9, 8192
    flat = np.full((B, 2, V), 0.75, np.float32)
    uni = np.zeros((B, 2), np.float32)
    uni[:, 0] = np.arange(B) * 2.0 ** -14  # r < 1 / 8192 or not
    uni[:, 1] = [0, 0.5, 0.25, 1 - 2.0 ** -13, 1 - 2.0 ** -24, 4096 / 8192, 4095 / 8192, 1 / 8192, 0.125]
    drafts = np.full((B, 1), 4095)
    got = run(ctx, flat, None, drafts, None, np.ones(B), uni)
    check(flat, None, drafts, None, np.ones(B), uni, got)
    assert list(got[1]) == [2, 2, 1, 1, 1, 1, 1, 1, 1]
    assert list(got[0][:2, 1]) == [0, 4096]


def test_temperatures(ctx):
    """Very cold, very warm and infinite temperatures."""
    rng = np.random.default_rng(7)
    for model in (False, True):
        logits, draft, drafts, temp, uni = inputs(rng, 6, 2, 6000, model)
        temp[:] = [1e-30, 1e-3, 50.0, 1e30, np.inf, 1e-45]
        logits[5] *= 1e30
        check(logits, draft, drafts, None, temp, uni, run(ctx, logits, draft, drafts, None, temp, uni), what=(model,))


@pytest.mark.parametrize("model", [False, True])
def test_numbers_outside_0_to_1(ctx, model):
    """Numbers that are no probabilities draw some entry of the row all the same, one with a weight."""
    rng = np.random.default_rng(71)
    logits, draft, drafts, temp, uni = inputs(rng, 8, 2, 5000, model)
    logits[:4] = np.where(np.arange(5000) == 4321, 3.0, -np.inf)
    drafts[:4] = 4321
    uni[:] = [[np.nan] * 3, [1, 1, 1], [2, -1, 5], [np.inf, 0.5, -np.inf]] * 2
    tokens, n, logp = run(ctx, logits, draft, drafts, None, temp, uni)
    assert np.all((n >= 1) & (n <= 3))
    for b in range(8):
        assert np.all((tokens[b, :n[b]] >= 0) & (tokens[b, :n[b]] < 5000)) and np.all(tokens[b, n[b]:] == -1)
        assert b >= 4 or np.all(tokens[b, :n[b]] == 4321)


@pytest.mark.parametrize("model", [False, True])
def test_the_tokens_have_the_targets_distribution(ctx, model):
    """The first token of 3 x 4096 sequences with drafts from another distribution: its counts are within 5 standard
    deviations of the target's probabilities."""
    rng = np.random.default_rng(8)
    V, B, temp = 6, 4096, np.float32(0.9)
    p_row, q_row = rng.standard_normal(V).astype(np.float32), rng.standard_normal(V).astype(np.float32)
    p, q = (probabilities(x, temp)[0] for x in (p_row, q_row))
    logits = np.broadcast_to(p_row, (B, 2, V)).copy()
    draft = np.broadcast_to(q_row, (B, 1, V)).copy() if model else None
    counts = np.zeros(V)
    for _ in range(3):
        drafts = rng.choice(V, (B, 1), p=q)
        if not model:
            drafts[:] = 2
        tokens, n, _ = run(ctx, logits, draft, drafts, None, np.full(B, temp), rng.random((B, 2), dtype=np.float32))
        assert np.all((n == 2) == (tokens[:, 1] >= 0))
        counts += np.bincount(tokens[:, 0], minlength=V)
    assert np.all(np.abs(counts - 3 * B * p) <= 5 * np.sqrt(3 * B * p * (1 - p))), (counts / (3 * B), p)


def test_calls_in_turn(ctx):
    """Calls of different sizes one after another without a wait, each three times with the same result."""
    rng = np.random.default_rng(9)
    jobs = []
    for B, T, V, model in ((3, 7, 30000, True), (1, 0, 5, False), (70, 2, 900, True), (2, 5, 128256, False)):
        x = inputs(rng, B, T, V, model)
        dev = [None if a is None else ctx.to_device(a) for a in (x[0], x[1], x[2].astype(np.int32), x[3], x[4])]
        outs = [[ctx.alloc(B * (T + 1) * 4), ctx.alloc(B * 4), ctx.alloc(B * (T + 1) * 4)] for _ in range(3)]
        jobs.append((B, T, V, x, dev, outs))
    for turn in range(3):
        for B, T, V, x, (lo, dr, d, t, u), outs in jobs:
            ctx.verify_drafts(lo, V, dr, V, V, B, T, d, None, t, u, *outs[turn])
    for B, T, V, x, dev, outs in jobs:
        got = [(o[0].download(np.int32, (B, T + 1)), o[1].download(np.int32, (B,)), o[2].download(np.float32, (B, T + 1))) for o in outs]
        check(x[0], x[1], x[2], None, x[3], x[4], got[0])
        for g in got[1:]:
            assert all(np.array_equal(a, b) for a, b in zip(g, got[0]))


# ---- together ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv", [Q8, F16])
def test_conversations_with_drafts(ctx, kv):
    """Three conversations of one attention layer over shared pages: prompts appended, then steps in which the pending token
    and its drafts are appended, attended, and the drafts judged by the layer's logits, a page added where one is full.
    Every step's attention is that of float64 over the cached values read back, and its tokens those of float64 judging
    the same logits."""
    rng = np.random.default_rng([51, kv])
    H, HKV, HD, V, page, T = 4, 2, 64, 500, 16, 3
    c = Pages(ctx, rng, kv, HKV, HD, page, [0, 0, 0], spare=40, n_table=8)
    free = list(rng.permutation(40))
    width = (H + 2 * HKV) * HD
    embed = rng.standard_normal((V, width)).astype(np.float32)
    head = (rng.standard_normal((H * HD, V)) * 0.6).astype(np.float32)
    cs = rope_angles(128, HD)
    lengths, pending = [0, 0, 0], [0, 0, 0]

    def room(b, n):
        while np.count_nonzero(c.table[b] >= 0) * page < n:
            c.table[b, np.count_nonzero(c.table[b] >= 0)] = free.pop()

    prompts = [rng.integers(0, V, n) for n in (21, 5, 47)]
    seq, pos = np.concatenate([[b] * len(p) for b, p in enumerate(prompts)]), np.concatenate([np.arange(len(p)) for p in prompts])
    for b, p in enumerate(prompts):
        room(b, len(p))
        lengths[b], pending[b] = len(p) - 1, int(p[-1])  # (the last one is the first step's pending token)
    c.table_dev = ctx.to_device(c.table)
    append(ctx, c, embed[np.concatenate(prompts)], seq, pos, H, HD, 1, cs)
    temp = np.array([0.8, 1.0, 0.0], np.float32)
    emitted = [[], [], []]
    for step in range(6):
        drafts = rng.integers(0, V, (3, T))
        n_draft = np.array([T, (step % 2) * T, T - 1])
        ids = np.concatenate([[[pending[b], *drafts[b]] for b in range(3)]])
        for b in range(3):
            room(b, lengths[b] + T + 1)
        c.table_dev = ctx.to_device(c.table)
        seq, pos = np.repeat(np.arange(3), T + 1), np.concatenate([np.arange(n, n + T + 1) for n in lengths])
        q = append(ctx, c, embed[ids.reshape(-1)], seq, pos, H, HD, 1, cs).reshape(3, T + 1, H, HD)
        n_keys = np.array([n + T + 1 for n in lengths], np.int32)
        out = ctx.alloc(q.nbytes)
        ctx.attn_paged(ctx.to_device(q), 3, T + 1, H, HKV, HD, *c.args, c.n_table, ctx.to_device(n_keys), 0, 0.125, out)
        got = out.download(np.float32, q.shape)
        every = [(b, p) for b in range(3) for p in range(n_keys[b])]
        rows = [ctx.alloc(len(every) * HKV * HD * 4) for _ in range(2)]
        s, p = np.array(every, np.int32).T
        ctx.kv_read_paged(len(every), ctx.to_device(np.ascontiguousarray(s)), ctx.to_device(np.ascontiguousarray(p)), HKV, HD,
                          *c.args, *c.table.shape, ts5hip.F32, *rows)
        k, v = (r.download(np.float32, (len(every), HKV, HD)).astype(np.float64) for r in rows)
        for b in range(3):
            for t in range(T + 1):
                for h in range(H):
                    kk, vv = (x[s == b][:lengths[b] + t + 1, h // 2] for x in (k, v))
                    e = kk @ q[b, t, h].astype(np.float64) * 0.125
                    w = np.exp(e - e.max())
                    want = w @ vv / w.sum()
                    assert np.linalg.norm(got[b, t, h] - want) <= 2e-6 * np.linalg.norm(want) + 1e-12
        logits = got.reshape(3, T + 1, H * HD) @ head
        if step % 3 == 2:  # drafts worth keeping
            drafts[:, 0] = logits[:, 0].argmax(-1)
        uni = rng.random((3, T + 1), dtype=np.float32)
        result = run(ctx, logits, None, drafts, n_draft, temp, uni)
        check(logits, None, drafts, n_draft, temp, uni, result, what=(step,))
        for b in range(3):
            new = list(result[0][b][:result[1][b]])
            emitted[b] += new
            lengths[b] += len(new)
            pending[b] = int(new[-1])
    assert all(len(e) >= 6 for e in emitted) and sum(map(len, emitted)) > 18


@pytest.mark.parametrize("V", [37, 4096, 20000, 151936])
def test_rows_equal_to_the_drafts(ctx, V):
    """Target and draft rows alike bit for bit, and a draft that is not kept (outside the vocabulary, or of probability 0 in both
    rows): p - q is 0 everywhere, and the token is drawn from p. The largest entry is shared by two places, and an entry in
    five has no probability."""
    rng = np.random.default_rng([10, V])
    B, T = 24, 2
    logits, draft, drafts, temp, uni = inputs(rng, B, T, V, True, noise=0.0)
    logits[:, :, [3, V - 2]] = 11.0
    logits[:, :, 1:V - 3:5] = -np.inf
    draft = logits[:, :T].copy()
    assert np.all(logits[:, :T, 1] == -np.inf)
    drafts[0::3, 0], drafts[1::3, 0], drafts[2::3, 0] = -1, V, 1
    temp[::4] = 1.0
    uni[:4, T], uni[4:8, T] = 0, 1 - 2.0 ** -24
    got = run(ctx, logits, draft, drafts, None, temp, uni)
    check(logits, draft, drafts, None, temp, uni, got)
    assert np.all(got[1] == 1)
