"""The entry points for drafted tokens without a GPU: refused arguments and
their reasons, counts of zero, and the host-side mask helpers."""
import ctypes as C
import os

import numpy as np
import pytest
from conftest import nb

P = 4096  # a non-null, aligned address that no refused call may touch


def rc(name, *args):
    """Status and reason of one call."""
    f = getattr(nb.lib(), name)
    return f(*args), nb.lib().nd_last_error().decode()


def refused(name, args, why):
    code, msg = rc(name, *args)
    assert code == 1, (name, args)  # cudaErrorInvalidValue
    assert msg.startswith(name + ":") and why in msg, msg


def rope_args(**kw):
    a = dict(x=P, ldx=96, y=P, ldy=96, pos=P, M=4, heads=2, dim=48, rot=48, theta=10000.0, inter=0, sc=None, inv=0)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("change,why", [
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(pos=None), "null"), (dict(M=-1), "negative"),
    (dict(heads=0), "heads"), (dict(dim=0), "heads"), (dict(heads=1 << 20, dim=48), "2^24"),
    (dict(rot=0), "rot_dim"), (dict(rot=7), "rot_dim"), (dict(rot=50), "rot_dim"),
    (dict(dim=300, rot=258, ldx=600, ldy=600), "rot_dim"),
    (dict(ldx=95), "stride"), (dict(ldy=95, y=2 * P), "stride"), (dict(ldy=97), "in place"),
    (dict(theta=0.0), "theta"), (dict(theta=float("nan")), "theta"), (dict(theta=float("inf")), "theta"),
    (dict(sc=nb.RopeScaling("linear", 0.0)), "factor"), (dict(sc=nb.RopeScaling("linear", float("nan"))), "factor"),
    (dict(sc=nb.RopeScaling("by_parts", 4.0)), "trained"),
    (dict(sc=nb.RopeScaling("by_parts", 4.0, trained=4096, fast=1.0, slow=1.0)), "fast"),
])
def test_rope_refusals(change, why):
    if change.get("sc") is not None:
        change = dict(change, sc=C.addressof(change["sc"]))
    refused("nd_rope", rope_args(**change), why)


def test_rope_refuses_an_unknown_scaling():
    s = nb.RopeScaling("linear", 2.0)
    s.kind = 3
    refused("nd_rope", rope_args(sc=C.addressof(s)), "kind")
    with pytest.raises(nb.NeedleError, match="unknown kind"):
        nb.RopeScaling("cubic")


def append_args(**kw):
    a = dict(k=P, ldk=96, v=P, ldv=128, sess=P, pos=P, M=4, int8=1, sessions=8, slots=16, kvh=2, qk=48, vh=64, kc=P,
             vc=P, ks=P, vs=P)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("change,why", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(pos=None), "null"), (dict(kc=None), "null"),
    (dict(vc=None), "null"), (dict(ks=None), "null"), (dict(vs=None), "null"), (dict(M=-3), "negative"),
    (dict(kvh=0), "kv_heads"), (dict(kvh=513), "kv_heads"), (dict(qk=0), "widths"), (dict(vh=257), "widths"),
    (dict(sessions=0), "sessions"), (dict(slots=0), "slots"), (dict(sess=None, M=9), "one row per session"),
    (dict(ldk=95), "stride"), (dict(ldv=127), "stride"),
])
def test_append_refusals(change, why):
    refused("nd_kv_append", append_args(**change), why)


def read_args(**kw):
    a = dict(kc=P, vc=P, ks=P, vs=P, int8=1, sessions=8, slots=16, kvh=2, qk=48, vh=64, sess=P, pos=P, M=4, k=P,
             ldk=96, v=P, ldv=128)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("change,why", [
    (dict(kc=None), "null"), (dict(vc=None), "null"), (dict(ks=None), "null"), (dict(vs=None), "null"),
    (dict(pos=None), "null"), (dict(k=None, v=None), "neither"), (dict(M=-1), "negative"), (dict(kvh=0), "kv_heads"),
    (dict(qk=257, ldk=514), "widths"), (dict(slots=0), "slots"), (dict(sess=None, M=9), "one row per session"),
    (dict(ldk=95), "stride"), (dict(ldv=127), "stride"),
])
def test_read_refusals(change, why):
    refused("nd_kv_read", read_args(**change), why)


def tree_args(**kw):
    a = dict(q=P, ldq=576, k=P, v=P, ks=P, vs=P, int8=1, slots=64, lo=P, hi=P, tk=P, tv=P, tks=P, tvs=P, mask=P, B=2,
             T=8, heads=12, kvh=2, qk=48, vh=64, out=P)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("change,why", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(ks=None), "null"),
    (dict(vs=None), "null"), (dict(lo=None), "null"), (dict(hi=None), "null"), (dict(out=None), "null"),
    (dict(tk=None), "draft"), (dict(tv=None), "draft"), (dict(tks=None), "scales"), (dict(tvs=None), "scales"),
    (dict(tk=None, tv=None), "mask without"), (dict(B=-1), "negative"), (dict(T=-1), "negative"),
    (dict(heads=11), "divide"), (dict(kvh=0), "kv_heads"), (dict(heads=0), "divide"), (dict(qk=46), "multiples of 4"),
    (dict(vh=132), "at most 128"), (dict(qk=0), "multiples"), (dict(T=4097), "4096"), (dict(slots=0), "slots"),
    (dict(slots=(1 << 30) + 1), "slots"), (dict(B=1 << 24), "2^30"), (dict(ldq=575), "ldq"), (dict(k=P + 2), "aligned"),
    (dict(tv=P + 1), "aligned"),
])
def test_tree_refusals(change, why):
    refused("nd_attend_tree", tree_args(**change), why)


def logits_args(**kw):
    a = dict(x=P, ld=100, rows=4, vocab=100, y=P, ldo=100, hist=P, off=P, gen=P, rep=P, pres=P, freq=P, bi=P, bv=P,
             bo=P, mask=P, mask_ld=4, masked=-1e9, picks=P)
    a.update(kw)
    return list(a.values()) + [None]


@pytest.mark.parametrize("change,why", [
    (dict(x=None), "null"), (dict(y=None), "null"), (dict(rows=-1), "negative"), (dict(vocab=0), "vocab"),
    (dict(ld=99), "stride"), (dict(ldo=99, y=2 * P), "stride"), (dict(ldo=104), "in place"), (dict(off=None), "offsets"),
    (dict(bv=None), "biases"), (dict(bo=None), "biases"), (dict(mask_ld=3), "mask_ld"),
])
def test_logits_refusals(change, why):
    refused("nd_logits_adjust", logits_args(**change), why)


def test_counts_of_zero_do_nothing():
    assert rc("nd_rope", *rope_args(M=0, x=None, y=None, pos=None))[0] == 0
    assert rc("nd_kv_append", *append_args(M=0, k=None, v=None, pos=None))[0] == 0
    assert rc("nd_kv_read", *read_args(M=0, kc=None, vc=None, pos=None))[0] == 0
    assert rc("nd_attend_tree", *tree_args(B=0, q=None))[0] == 0
    assert rc("nd_attend_tree", *tree_args(T=0, q=None))[0] == 0
    assert rc("nd_logits_adjust", *logits_args(rows=0, x=None))[0] == 0


def test_tree_mask_names_ancestors():
    parents = [-1, 0, 0, 1, -1, 4, 3]
    m = nb.tree_mask(parents)
    assert m.shape == (7, 1) and m.dtype == np.uint32
    for t in range(7):
        want, p = 0, t
        while p >= 0:
            want |= 1 << p
            p = parents[p]
        assert int(m[t, 0]) == want
    chain = nb.tree_mask([t - 1 for t in range(70)])
    assert chain.shape == (70, 3)
    for t in range(70):
        got = sum(int(w) << (32 * i) for i, w in enumerate(chain[t]))
        assert got == (1 << (t + 1)) - 1
    for bad in ([0], [-1, 2], [-2]):
        with pytest.raises(nb.NeedleError):
            nb.tree_mask(bad)


def test_pack_mask_takes_truth_and_grammar_masks():
    rng = np.random.default_rng(0)
    for n in (1, 31, 32, 33, 500):
        keep = rng.random((3, n)) < 0.4
        w = nb.pack_mask(keep)
        assert w.shape == (3, (n + 31) // 32) and w.dtype == np.uint32
        for r in range(3):
            for i in range(n):
                assert bool((int(w[r, i // 32]) >> (i % 32)) & 1) == bool(keep[r, i])
        assert np.array_equal(nb.pack_mask(np.where(keep, 0.0, -1e9).astype(np.float32)), w)


def test_the_workload_file_runs_here():
    """Cases, draws and work figures of perf/operators.py are plain values."""
    import importlib.util
    import random
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("draft_workloads", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    names = [c["name"] for c in m.listed()]
    assert len(set(names)) == len(names) and 4 <= len(names) <= 12
    rng = random.Random(1)
    for c in m.listed() + [m.draw(rng) for _ in range(60)]:
        w = m.work(c)
        assert w["bytes"] > 0 and w["flops"] > 0
