"""What the entry points around a KV cache (trees, key weights, eviction, block-sparse attention) refuse, on the
CPU: their arguments are checked before their context, so a null context reaches every check and no GPU."""
import ctypes

import pytest

from tokenstation5_amd import ts5hip

L = ts5hip.lib
P, Q = 1 << 20, 1 << 24  # addresses that are never read
ARG, UNS = ts5hip.ERR_ARG, ts5hip.ERR_UNSUPPORTED
Q8, F16 = ts5hip.KV_Q8, ts5hip.KV_F16

CALLS = {
    "append": ("ts5hip_rope_kv_append_at", dict(
        ctx=None, qkv=P, ntok=3, pos=P, slot0=P, H=8, HKV=2, HD=128, n_rot=128, neox=0, cs=P, n_pos=64, n_ctx=256, kv=Q8,
        bias=None, q_norm=None, k_norm=None, eps=1e-6, q_out=P, k=P, ks=P, v=P, vs=P)),
    "tree": ("ts5hip_attn_tree", dict(
        ctx=None, q=P, B=1, T=8, H=8, HKV=2, HD=128, kv=Q8, k=P, ks=P, v=P, vs=P, n_ctx=256, n_past=P, mask=P, scale=0.1,
        out=P)),
    "path": ("ts5hip_kv_path", dict(
        ctx=None, B=1, HKV=2, HD=128, kv=Q8, k=P, ks=P, v=P, vs=P, n_ctx=256, slots=P, n=5, slot0=P)),
    "weights": ("ts5hip_attn_decode_weights", dict(
        ctx=None, q=P, B=1, H=8, HKV=2, HD=128, kv=Q8, k=P, ks=P, v=P, vs=P, n_ctx=256, n_keys=P, scale=0.1, out=P, acc=P,
        acc_out=P)),
    "prompt": ("ts5hip_attn_prompt_weights", dict(
        ctx=None, q=P, nq=16, H=8, HKV=2, HD=128, kv=Q8, k=P, ks=P, v=P, vs=P, n_ctx=256, pos0=100, scale=0.1, out=P, acc=P,
        acc_out=P)),
    "evict": ("ts5hip_kv_evict", dict(
        ctx=None, B=1, HKV=2, HD=128, kv=Q8, k=P, ks=2 * P, v=3 * P, vs=4 * P, n_ctx=256, n_keys=P, acc=5 * P, n_keep=100,
        n_first=4, n_last=64, n_ctx_out=128, k_out=6 * P, ks_out=7 * P, v_out=8 * P, vs_out=9 * P, acc_out=10 * P, kept=P,
        n_out=None)),
    "bounds": ("ts5hip_kv_block_bounds", dict(
        ctx=None, B=1, HKV=2, HD=128, kv=Q8, k=P, ks=P, n_ctx=256, n_keys=P, n_new=5, block=64, bounds=P)),
    "sparse": ("ts5hip_attn_sparse", dict(
        ctx=None, q=P, B=1, H=8, HKV=2, HD=128, kv=Q8, k=P, ks=P, v=P, vs=P, n_ctx=256, n_keys=P, per=1, bounds=P, block=64,
        n_pick=4, scale=0.1, out=P, picked=None)),
}
NEED = dict(append="qkv pos slot0 cs q_out k ks v vs", tree="q k ks v vs n_past mask out", path="k ks v vs slots slot0",
            weights="q k ks v vs n_keys out acc acc_out", prompt="q k ks v vs out acc acc_out",
            evict="k ks v vs n_keys acc k_out ks_out v_out vs_out acc_out kept", bounds="k ks n_keys bounds",
            sparse="q k ks v vs n_keys bounds out")
SHAPES = [dict(HD=96), dict(HD=32), dict(kv=ts5hip.KV_F32), dict(kv=7), dict(HKV=0), dict(n_ctx=0), dict(HKV=513),
          dict(n_ctx=1 << 25), dict(k=P + 8), dict(ks=P + 2)]
OWN = {
    "append": [dict(ntok=0), dict(ntok=4097), dict(n_rot=130), dict(n_rot=63), dict(n_pos=0), dict(H=7), dict(v=P + 8)],
    "tree": [dict(T=0), dict(T=65), dict(T=20, n_ctx=19), dict(B=0), dict(B=4097), dict(H=7), dict(H=34), dict(q=P + 4),
             dict(out=P + 8), dict(mask=P + 4), dict(vs=P + 1)],
    "path": [dict(n=0), dict(n=65), dict(B=0)],
    "weights": [dict(B=0), dict(H=9), dict(H=0), dict(q=P + 8), dict(out=P + 4)],
    "prompt": [dict(nq=0), dict(nq=4097, n_ctx=8192), dict(pos0=-1), dict(pos0=241), dict(pos0=2**31 - 1), dict(H=7),
               dict(nq=4096, n_ctx=8192, H=1024, HKV=64)],
    "evict": [dict(n_keep=0), dict(n_keep=129), dict(n_first=-1), dict(n_last=-1), dict(n_first=50, n_last=51),
              dict(n_first=2**31 - 1, n_last=1), dict(k_out=P), dict(k_out=P + 1024), dict(acc_out=5 * P + 16),
              dict(v_out=P), dict(vs_out=2 * P), dict(k_out=None), dict(n_ctx_out=0)],
    "bounds": [dict(block=0), dict(block=48), dict(block=256), dict(n_new=0), dict(n_new=-3), dict(bounds=P + 8), dict(B=0)],
    "sparse": [dict(block=20), dict(n_pick=0), dict(n_pick=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
               dict(B=0), dict(H=7), dict(H=34), dict(bounds=P + 8), dict(q=P + 8), dict(out=P + 8), dict(B=2049)],
}


def call(name, **change):
    f, args = CALLS[name]
    rc = getattr(L(), f)(*dict(args, **change).values())
    return rc, L().ts5hip_last_error(None).decode()


@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_reach_the_context(name):
    assert call(name) == (ARG, "ctx is null")
    if "kv" in CALLS[name][1]:  # an f16 cache needs no scales
        none = {a: None for a in ("ks", "vs", "ks_out", "vs_out") if a in CALLS[name][1]}
        assert call(name, kv=F16, **none) == (ARG, "ctx is null")


@pytest.mark.parametrize("name,arg", [(n, a) for n, args in NEED.items() for a in args.split()])
def test_null_arguments(name, arg):
    assert call(name, **{arg: None}) == (ARG, "null argument")


@pytest.mark.parametrize("name,change", [(n, c) for n in CALLS for c in SHAPES] + [(n, c) for n, cs in OWN.items() for c in cs])
def test_refused(name, change):
    rc, text = call(name, **change)
    assert rc in (ARG, UNS) and text not in ("ctx is null", ""), (rc, text)


def test_bounds_bytes():
    f = L().ts5hip_kv_bounds_bytes
    assert f(3, 8, 128, 1000, 64) == 3 * 8 * 16 * 2 * 128 * 2
    assert f(1, 1, 64, 1, 128) == 256
    assert f(1, 1, 64, 2 ** 31 - 1, 128) == 2 ** 24 * 256
    assert [f(*a) for a in ((0, 1, 64, 1, 64), (1, 0, 64, 1, 64), (1, 1, 64, 0, 64), (1, 1, 64, 1, 8))] == [-1] * 4


@pytest.mark.parametrize("H,HKV,HD", [(14, 2, 64), (5, 1, 128), (32, 8, 128), (6, 2, 256)])
@pytest.mark.parametrize("nq,keys", [(1, 1), (5, 700), (37, 4096), (530, 1631)])
def test_prompt_weights_scratch_is_aligned(H, HKV, HD, nq, keys):
    """The parts of the prompt key weights' scratch begin on lines of their own, none inside another, whatever the rows."""
    layout = L()._ZN6ts5hip26attn_prompt_weights_layoutEiiiiiiiPm
    layout.argtypes, layout.restype = [ctypes.c_int] * 7 + [ctypes.POINTER(ctypes.c_size_t)], None
    total = L()._ZN6ts5hip33attn_prompt_weights_scratch_bytesEiiiiiii
    total.argtypes, total.restype = [ctypes.c_int] * 7, ctypes.c_size_t
    for f16 in (0, 1):
        at = (ctypes.c_size_t * 4)()
        layout(nq, H, HKV, HD, f16, keys, 256, at)
        assert all(x % 256 == 0 for x in at), list(at)
        tiles = -(-nq * (H // HKV) // 16)
        ends = [at[0] + HKV * tiles * (HD // 32) * 2 * 64 * 16, at[1] + HKV * tiles * 16 * 4, at[2] + H * nq * 4]
        assert all(e <= b for e, b in zip(ends, list(at)[1:])) and at[3] <= total(nq, H, HKV, HD, f16, keys, 256)


@pytest.mark.parametrize("change", [dict(n_out=P), dict(n_keys=11 * P, n_out=11 * P), dict(n_keys=11 * P, n_out=11 * P + 4, B=3),
                                    dict(n_out=3 * P + 4096), dict(n_out=5 * P), dict(n_out=10 * P), dict(n_out=6 * P + 64),
                                    dict(n_keys=6 * P + 8), dict(n_keys=10 * P), dict(v_out=6 * P), dict(vs_out=7 * P + 512)])
def test_evict_outputs_of_their_own(change):
    """Counts written over the counts that other workgroups still read, and outputs over inputs or other outputs."""
    assert call("evict", **change) == (ARG, "an eviction's outputs lie over its inputs or each other")
    assert call("evict", n_keys=12 * P, n_out=11 * P) == (ARG, "ctx is null")


@pytest.mark.parametrize("name,B", [("weights", 1), ("weights", 3), ("prompt", 1)])
def test_sums_over_themselves(name, B):
    """acc_out beside acc or acc itself, not a part of it: one thread would write what another has yet to read."""
    more = dict(B=B) if name == "weights" else {}
    size = B * 2 * 256 * 4
    for at in (4, 1024, size - 4, -4, 4 - size):
        assert call(name, acc=Q, acc_out=Q + at, **more) == (ARG, "acc_out is acc or does not overlap it")
    for at in (0, size, -size):
        assert call(name, acc=Q, acc_out=Q + at, **more) == (ARG, "ctx is null")
