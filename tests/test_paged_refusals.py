"""What the entry points around caches in pages and the verification of drafts refuse, on the CPU: their arguments are
checked before their context, so a null context reaches every check and no GPU."""
import pytest

from tokenstation5_amd import ts5hip

L = ts5hip.lib
P = 1 << 26  # addresses that are never read
ARG, UNS = ts5hip.ERR_ARG, ts5hip.ERR_UNSUPPORTED
Q8, F16 = ts5hip.KV_Q8, ts5hip.KV_F16
POOL = dict(kv=Q8, k=P, ks=2 * P, v=3 * P, vs=4 * P, n_pages=9, page=64, table=5 * P)

CALLS = {
    "append": ("ts5hip_rope_kv_append_paged", dict(
        ctx=None, qkv=7 * P, ntok=3, seq=P, pos=P, H=8, HKV=2, HD=128, n_rot=128, neox=0, cs=P, n_pos=64, bias=None, q_norm=None,
        k_norm=None, eps=1e-6, q_out=6 * P, **POOL, n_seq=2, n_table=4)),
    "read": ("ts5hip_kv_read_paged", dict(
        ctx=None, ntok=3, seq=P, pos=P, HKV=2, HD=128, **POOL, n_seq=2, n_table=4, out_type=0, k_out=6 * P, v_out=7 * P)),
    "attn": ("ts5hip_attn_paged", dict(
        ctx=None, q=6 * P, B=2, n_new=1, H=8, HKV=2, HD=128, **POOL, n_table=4, n_keys=P, window=0, scale=0.1, out=7 * P)),
    "verify": ("ts5hip_verify_drafts", dict(
        ctx=None, logits=P, ld=1000, draft=2 * P, ld_draft=1000, V=1000, B=2, T=5, drafts=3 * P, n_draft=4 * P, temp=5 * P,
        uni=6 * P, tokens=7 * P, n_tokens=8 * P, logp=9 * P)),
}
NEED = dict(append="qkv seq pos cs q_out k ks v vs table", read="seq pos k ks v vs table k_out v_out",
            attn="q k ks v vs table n_keys out", verify="logits drafts temp uni tokens n_tokens")
PAGED = ("append", "read", "attn")
SHAPES = [dict(HD=96), dict(HD=32), dict(kv=ts5hip.KV_F32), dict(kv=7), dict(HKV=0), dict(HKV=513), dict(k=P + 8),
          dict(v=P + 4), dict(ks=P + 2), dict(page=0), dict(page=8), dict(page=48), dict(page=512), dict(page=-64),
          dict(n_pages=0), dict(n_pages=-1), dict(n_table=0), dict(n_table=-3), dict(n_table=(1 << 24) + 1)]
OWN = {
    "append": [dict(ntok=0), dict(ntok=65536), dict(n_rot=130), dict(n_rot=63), dict(n_rot=-2), dict(n_pos=0), dict(H=7),
               dict(n_seq=0), dict(q_out=6 * P + 8), dict(qkv=7 * P + 4), dict(bias=P + 4), dict(q_norm=P + 8),
               dict(k_norm=P + 4), dict(cs=P + 8), dict(q_out=7 * P), dict(q_out=7 * P + 3 * 12 * 512 - 16),
               dict(q_out=7 * P - 3 * 8 * 512 + 16), dict(q_out=P), dict(q_out=5 * P), dict(q_out=4 * P + 1024)],
    "read": [dict(ntok=0), dict(ntok=(1 << 24) + 1), dict(n_seq=0), dict(out_type=2), dict(out_type=-1), dict(k_out=6 * P + 8),
             dict(v_out=6 * P), dict(v_out=6 * P + 3 * 2 * 512 - 16), dict(k_out=P), dict(v_out=2 * P), dict(k_out=4 * P + 1024),
             dict(v_out=5 * P)],
    "attn": [dict(B=0), dict(B=4097), dict(n_new=0), dict(n_new=17), dict(H=7), dict(H=34), dict(window=-1), dict(q=6 * P + 4),
             dict(out=7 * P + 8), dict(out=6 * P), dict(out=6 * P + 2 * 8 * 512 - 16), dict(B=4096, n_table=1 << 17),
             dict(out=P), dict(out=3 * P + 1024), dict(out=4 * P), dict(out=5 * P)],
    "verify": [dict(V=0), dict(V=(1 << 20) + 1, ld=1 << 21, ld_draft=1 << 21), dict(ld=999), dict(ld_draft=999), dict(B=0),
               dict(B=4097), dict(T=-1), dict(T=64), dict(ld=1 << 41), dict(tokens=3 * P), dict(tokens=P), dict(n_tokens=4 * P),
               dict(n_tokens=7 * P + 4), dict(logp=7 * P), dict(logp=6 * P + 8), dict(tokens=P + 4 * (2 * 6 * 1000 - 1)),
               dict(tokens=2 * P + 4 * (2 * 5 * 1000 - 1))],
}


def call(name, **change):
    f, args = CALLS[name]
    rc = getattr(L(), f)(*dict(args, **change).values())
    return rc, L().ts5hip_last_error(None).decode()


@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_reach_the_context(name):
    assert call(name) == (ARG, "ctx is null")


@pytest.mark.parametrize("name,change", [(n, dict(kv=F16, ks=None, vs=None)) for n in PAGED] + [
    ("append", dict(bias=P, q_norm=P, k_norm=P, n_rot=0)), ("append", dict(ntok=65535, q_out=90 * P)), ("read", dict(out_type=1)),
    ("read", dict(ntok=1 << 24, k_out=100 * P, v_out=2000 * P)), ("attn", dict(n_new=16, window=2 ** 31 - 1)),
    ("attn", dict(n_table=1 << 24)), ("attn", dict(B=4096, n_table=1 << 16, out=70 * P)), ("verify", dict(draft=None, ld_draft=0)),
    ("verify", dict(T=0, drafts=None, draft=None)), ("verify", dict(n_draft=None, logp=None)),
    ("verify", dict(V=1, B=4096, T=63, draft=None, ld=1, logits=P))])
def test_other_good_arguments(name, change):
    assert call(name, **change) == (ARG, "ctx is null")


@pytest.mark.parametrize("name,arg", [(n, a) for n, args in NEED.items() for a in args.split()])
def test_null_arguments(name, arg):
    assert call(name, **{arg: None}) == (ARG, "null argument")


@pytest.mark.parametrize("name,change", [(n, c) for n in PAGED for c in SHAPES] + [(n, c) for n, cs in OWN.items() for c in cs])
def test_refused(name, change):
    rc, text = call(name, **change)
    assert rc in (ARG, UNS) and text not in ("ctx is null", ""), (rc, text)


@pytest.mark.parametrize("change", [
    # q_out over the biases (12 heads of 128), the norms (128) and the angles (64 positions of 128): their first and last bytes
    dict(bias=6 * P), dict(bias=6 * P - 12 * 512 + 16), dict(q_norm=6 * P + 3 * 8 * 512 - 16), dict(q_norm=6 * P - 512 + 16),
    dict(k_norm=6 * P), dict(k_norm=6 * P - 512 + 16), dict(cs=6 * P + 16), dict(cs=6 * P - 64 * 512 + 16),
    # the pool (9 pages of 2 x 64 rows of 128 bytes, 8 of scales) over its own parts, the new rows and the table
    dict(v=P), dict(v=P + 9 * 128 * 128 - 16), dict(ks=P + 1024), dict(vs=2 * P + 9 * 128 * 8 - 4), dict(vs=3 * P),
    dict(k=7 * P), dict(v=7 * P + 3 * 12 * 512 - 16), dict(ks=7 * P), dict(vs=7 * P + 16), dict(k=5 * P), dict(vs=5 * P + 4),
    dict(table=3 * P + 16), dict(kv=F16, ks=None, vs=None, v=P + 9 * 128 * 256 - 16)])
def test_appends_over_what_they_read_or_write(change):
    rc, text = call("append", **change)
    assert (rc, text) == (ARG, "outputs lie over inputs or each other")


@pytest.mark.parametrize("change", [
    dict(bias=6 * P - 12 * 512), dict(bias=6 * P + 3 * 8 * 512), dict(q_norm=6 * P - 512), dict(k_norm=6 * P + 3 * 8 * 512),
    dict(cs=6 * P - 64 * 512), dict(cs=6 * P, n_rot=0), dict(v=P + 9 * 128 * 128), dict(ks=P + 9 * 128 * 128),
    dict(kv=F16, ks=P, vs=P), dict(k=7 * P + 3 * 12 * 512)])
def test_appends_beside_what_they_read_or_write(change):
    assert call("append", **change) == (ARG, "ctx is null")
