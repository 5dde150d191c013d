"""Where the operators for drafted tokens can go wrong: nd_attend_tree with many
rows of a KV head (the tcgen05 form) over odd lengths, far apart value scales,
hidden and seen garbage; the int8 writer on special values; nd_logits_adjust
with long bias lists and vocabularies of several turns; two host threads.

Tolerances are those of the 64-bit references (Tree.want, LOGIT_TOL), derived
there.
"""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
from conftest import ROOT, nb
from test_gpu_draft import LOGIT_TOL, Tree, all_calls, dev, logits_ref, ptr, quant_ref

pytestmark = pytest.mark.gpu

# More than 16 rows (T * heads / kv_heads) of a KV head, aligned widths.
MANY_ROWS = [
    # B, T, heads, kv_heads, qk, vh, slots, ctx
    (1, 17, 1, 1, 16, 16, 1, 1),         # one ring place
    (2, 9, 2, 1, 48, 64, 63, 63),        # a step short of one block
    (1, 3, 16, 2, 48, 64, 65, 64),
    (2, 43, 3, 1, 64, 64, 200, 129),     # 129 rows: a second tile of one row
    (1, 127, 2, 1, 32, 32, 150, 90),     # 254 rows
    (1, 32, 8, 2, 48, 48, 1000, 990),
    (1, 20, 8, 1, 64, 32, 4200, 4111),   # split over the positions, partial results joined
    (2, 5, 16, 2, 128, 128, 300, 255),
    (1, 65, 4, 2, 128, 64, 129, 127),    # 130 rows, three mask words
    (1, 6, 8, 2, 80, 64, 500, 431),
    (2, 6, 12, 4, 16, 128, 70, 0),       # the draft alone
    (1, 24, 4, 1, 112, 16, 2500, 2477),
    (1, 8, 32, 8, 128, 128, 3000, 2999),
]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("shape", MANY_ROWS)
def test_many_rows_match_64_bits(cuda, int8, shape):
    B, T, heads, kvh, qk, vh, slots, ctx = shape
    Tree(B, T, heads, kvh, qk, vh, slots, ctx, int8, seed=sum(shape), extra=T % 4).check(cuda)


@pytest.mark.parametrize("int8", [False, True])
def test_many_nodes_of_a_chain(cuda, int8):
    """Hundreds of nodes: several row tiles and mask words."""
    Tree(1, 300, 2, 1, 48, 64, 40, 33, int8, seed=2, mask="chain").check(cuda)
    Tree(1, 130, 3, 3, 16, 16, 40, 33, int8, seed=3).check(cuda)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,heads,kvh,qk,vh", [(5, 8, 2, 48, 64), (12, 4, 2, 128, 128)])
def test_many_rows_over_value_scales_far_apart(cuda, int8, T, heads, kvh, qk, vh):
    """Blocks of values 2^12 and more apart: rows that see small ones alone keep
    their accuracy, as do rows that see all."""
    torch = cuda
    c = Tree(2, T, heads, kvh, qk, vh, 640, 640, int8, seed=6)
    for i, s in enumerate([1e-30, 1e-3, 1e12, 1e-12, 1.0, 1e20, 1e-20, 1e3, 1e-38, 1e18]):
        at = slice(64 * i + 7, 64 * i + 71)
        if int8:
            c.vs[:, at] *= np.float32(s)
        else:
            c.v[:, at] *= np.float32(s)
    c.check(torch)
    # nodes with windows of a few positions each, in blocks of every size
    r = np.random.default_rng(0)
    c.mask[:] = 0
    for b in range(2):
        for t in range(T):
            first = int(r.integers(0, 600))
            c.lo[b, t], c.hi[b, t] = first, first + int(r.integers(0, 40))
    c.check(torch)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("gain", [(1e-6, 1e-8), (6.0, 3e4), (1e4, 1.0), (1e-20, 1e30)])
def test_many_rows_over_the_range_of_values(cuda, int8, gain):
    Tree(2, 11, 12, 2, 48, 64, 90, 80, int8, seed=5, qgain=gain[0], vgain=gain[1]).check(cuda)
    Tree(1, 11, 8, 2, 128, 128, 90, 80, int8, seed=5, qgain=gain[0], vgain=gain[1]).check(cuda)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), -3.4028234663852886e38])
def test_hidden_garbage_never_reaches_many_rows(cuda, int8, wide, bad):
    """Ring places out of range and a node nobody sees hold garbage."""
    torch = cuda
    qk, vh = (128, 128) if wide else (48, 64)
    c = Tree(2, 20, 8, 2, qk, vh, 200, 130, int8, seed=23)
    c.mask &= ~np.uint32(1 << 11)
    c.mask[:, 11] = np.uint32(1 << 11)
    want, tol = c.want()
    for b in range(2):
        seen = set(s for t in range(20) for s in c.seen(b, t)[0])
        free = [s for s in range(200) if s not in seen]
        assert free
        if int8:
            c.ks[b, free] = c.vs[b, free] = bad
            c.tks[b, 11] = c.tvs[b, 11] = bad
        else:
            c.k[b, free] = c.v[b, free] = bad
            c.tk[b, 11] = c.tv[b, 11] = bad
        c.q[b, 11] = bad
    others = [t for t in range(20) if t != 11]
    got = c.run(torch).cpu().numpy()
    assert np.all(np.abs(got - want)[:, others] <= tol[:, others])


@pytest.mark.parametrize("wide", [False, True])
def test_a_seen_value_that_is_not_finite_reaches_its_dimension(cuda, wide):
    torch = cuda
    qk, vh = (128, 128) if wide else (48, 64)
    d = Tree(1, 9, 8, 2, qk, vh, 70, 40, False, seed=2)
    want, tol = d.want()
    ring, _ = d.seen(0, 0)
    hit = np.zeros(want.shape, bool)
    hit[0, :, :4, 5] = True
    for bad in (float("nan"), float("inf")):
        d.v[0, ring[3], 0, 5] = bad
        got = d.run(torch).cpu().numpy()
        assert np.array_equal(got[hit], np.full(hit.sum(), bad, np.float32), equal_nan=True)
        assert np.all((np.abs(got - want) <= tol)[~hit])


@pytest.mark.parametrize("int8", [False, True])
def test_many_rows_with_windows_and_empty_nodes(cuda, int8):
    torch = cuda
    c = Tree(3, 12, 12, 2, 48, 64, 70, 60, int8, seed=9)
    for t in range(12):
        c.lo[:, t] += 4 * t
    c.lo[0, 3], c.hi[0, 3] = 5, 4
    c.mask[0, 3] = 0
    c.lo[1, :], c.hi[1, :] = 0, 2000
    c.lo[2, 0], c.hi[2, 0] = 3, 9
    c.lo[2, 1], c.hi[2, 1] = 100000, 100020
    c.lo[2, 2], c.hi[2, 2] = 2147483647 - 20, 2147483647
    c.lo[2, 3], c.hi[2, 3] = -50, 12
    c.lo[2, 4], c.hi[2, 4] = -2147483648, -20
    got = c.check(torch)
    assert np.all(got[0, 3] == 0.0)
    c.hi[:] = -1
    c.mask[:] = 0
    assert np.all(c.check(torch) == 0.0)


@pytest.mark.parametrize("shape", [(1, 4, 1, 128, 128, 5651), (2, 4, 1, 32, 32, 6007), (1, 12, 2, 48, 64, 9001),
                                   (9, 4, 1, 128, 128, 5651), (4, 12, 2, 48, 64, 9001)])
@pytest.mark.parametrize("int8", [False, True])
def test_long_contexts_are_as_exact_as_32_bits(cuda, int8, shape):
    """Sums over thousands of positions lose no more than the same sums in plain
    32-bit products and additions: nothing is left to accumulators that truncate."""
    torch = cuda
    T, heads, kvh, qk, vh, ctx = shape
    c = Tree(1, T, heads, kvh, qk, vh, ctx, ctx, int8, seed=ctx)
    c.lo[:] = 0
    c.hi[:] = ctx - 1
    c.mask[:] = 0
    got = c.run(torch).cpu().numpy()[0]
    k, v = c.k[0].astype(np.float64), c.v[0].astype(np.float64)
    if int8:
        k, v = k * c.ks[0][..., None], v * c.vs[0][..., None]
    q = c.q[0, :, : heads * qk].reshape(T, heads, qk)

    def attend(dt):
        out = np.zeros((T, heads, vh), dt)
        for h in range(heads):
            kh, vv = k[:, h // (heads // kvh)].astype(dt), v[:, h // (heads // kvh)].astype(dt)
            s = torch.from_numpy(q[:, h].astype(dt)).cuda() @ torch.from_numpy(kh).cuda().T / np.sqrt(qk)
            w = torch.exp(s - s.max(-1, keepdim=True).values)
            out[:, h] = (w @ torch.from_numpy(vv).cuda() / w.sum(-1, keepdim=True)).cpu().numpy()
        return out

    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    want, plain = attend(np.float64), attend(np.float32)
    torch.backends.cuda.matmul.allow_tf32 = old
    far = lambda x: float(np.linalg.norm(x - want) / np.linalg.norm(want))  # noqa: E731
    assert far(got) <= max(1.5 * far(plain), 2.0 ** -20), (far(got), far(plain))


@pytest.mark.parametrize("int8", [False, True])
def test_outputs_at_any_float(cuda, int8):
    """An output start that is 4-byte aligned only, guarded on both sides."""
    torch = cuda
    c = Tree(2, 8, 6, 2, 48, 64, 90, 80, int8, seed=8)
    c.check(torch)
    want, tol = c.want()
    n = want.size
    buf = torch.full((n + 6,), 7.0, device="cuda")
    c.call(c.keep, buf[3:])
    got = buf.cpu().numpy()
    assert np.all(got[:3] == 7.0) and np.all(got[3 + n:] == 7.0)
    assert np.all(np.abs(got[3: 3 + n].reshape(want.shape) - want) <= tol)


def test_many_rows_past_32_bit_offsets(cuda):
    """The last places of a ring of more than 2^31 codes."""
    torch = cuda
    S, slots, d = 2, 1 << 24, 128
    kc, vc = (torch.zeros(S, slots, 1, d, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(S, slots, 1, device="cuda") for _ in range(2))
    vc[1, -100:] = torch.randint(-127, 128, (100, 1, d), dtype=torch.int8, device="cuda")
    T = 20
    q = torch.zeros(S, T, 1, d, device="cuda")
    hi = torch.full((S, T), slots - 1, dtype=torch.int32, device="cuda")
    lo = hi - 99
    out = torch.zeros(S, T, 1, d, device="cuda")
    nb.attend_tree(ptr(q), d, ptr(kc), ptr(vc), ptr(ks), ptr(vs), True, slots, ptr(lo), ptr(hi), None, None, None, None,
                   None, S, T, 1, 1, d, d, ptr(out))
    want = vc[1, -100:, 0].double().mean(0)  # equal scores
    # weights of 1: sums of whole numbers below 2^24, one division
    assert torch.all(out[0] == 0) and torch.all((out[1, :, 0].double() - want).abs() <= 2.0 ** -20 * 127)


# ------------------------------------------------------------------ int8 codes
@pytest.mark.parametrize("d,vh", [(48, 64), (128, 32), (20, 36), (7, 9)])
def test_append_of_special_vectors_equals_the_standalone_quantiser(cuda, d, vh):
    """Zeros, denormals, the largest floats, exact halves: the codes and scales
    of nd_kv_quant to the bit."""
    torch = cuda
    r = np.random.default_rng(1)
    M = 24
    x = (r.normal(size=(M, d + vh))).astype(np.float32)
    x[0] = 0.0
    x[1] = -0.0
    x[2] *= np.float32(1e-39)               # denormal values and scales
    x[3] = np.float32(1e-45)
    with np.errstate(over="ignore"):
        x[4] *= np.float32(1e38)
    x[5] = np.float32(3.4028234e38)
    x[6] = -np.float32(3.4028234e38)
    x[7] = r.integers(-254, 255, d + vh) / np.float32(2)   # halves on the way to the codes
    x[7, 0] = x[7, d] = 127.0
    x[8] = np.where(r.random(d + vh) < 0.5, 1.0, -1.0)
    x[9, :] = 0.0
    x[9, d - 1] = x[9, d + vh - 1] = -2.5
    x[10] = np.nextafter(np.float32(0.5), np.float32(0), dtype=np.float32)
    x[10, 0] = x[10, d] = 127.0
    xd = dev(torch, x)
    kc, vc = (torch.zeros(M, 1, 1, n, dtype=torch.int8, device="cuda") for n in (d, vh))
    ks, vs = (torch.zeros(M, 1, 1, device="cuda") for _ in range(2))
    pos = torch.zeros(M, dtype=torch.int32, device="cuda")
    sess = torch.arange(M, dtype=torch.int32, device="cuda")
    nb.kv_append(ptr(xd), d + vh, ptr(xd) + 4 * d, d + vh, ptr(sess), ptr(pos), M, True, M, 1, 1, d, vh, ptr(kc), ptr(vc),
                 ptr(ks), ptr(vs))
    for at, n, codes, scales in ((0, d, kc, ks), (d, vh, vc, vs)):
        part = xd[:, at: at + n].contiguous()
        if n > 64:  # wider than nd_kv_quant takes: its steps on the host, of finite vectors
            ok = np.isfinite(x[:, at: at + n]).all(1)
            with np.errstate(all="ignore"):
                wc, ws = quant_ref(x[ok, at: at + n])
            assert np.array_equal(scales.cpu().numpy().reshape(-1)[ok], ws)
            assert np.array_equal(codes.cpu().numpy().reshape(M, n)[ok], wc)
            continue
        q, sc = torch.zeros(M, n, dtype=torch.int8, device="cuda"), torch.zeros(M, device="cuda")
        nb.kv_quant(ptr(part), M, n, ptr(q), ptr(sc))
        assert torch.equal(sc, scales.reshape(-1))
        assert torch.equal(q, codes.reshape(M, n)), torch.nonzero(q != codes.reshape(M, n))[:4]


def test_append_at_the_largest_positions(cuda):
    """A row near the last position keeps its place: the row a ring's length
    behind it in the call is skipped, not its successor."""
    torch = cuda
    M, slots = 9, 8
    x = torch.randn(M, 32, device="cuda")
    pos = torch.full((M,), -1, dtype=torch.int32, device="cuda")
    pos[0], pos[8] = 2147483644, -2147483644  # 8 apart modulo 2^32
    sess = torch.zeros(M, dtype=torch.int32, device="cuda")
    for int8 in (False, True):
        dt = torch.int8 if int8 else torch.float32
        kc, vc = (torch.zeros(1, slots, 1, 16, dtype=dt, device="cuda") for _ in range(2))
        ks, vs = (torch.zeros(1, slots, 1, device="cuda") for _ in range(2)) if int8 else (None, None)
        nb.kv_append(ptr(x), 32, ptr(x) + 64, 32, ptr(sess), ptr(pos), M, int8, 1, slots, 1, 16, 16, ptr(kc), ptr(vc),
                     ptr(ks), ptr(vs))
        want = quant_ref(x[:1, :16].cpu().numpy())[0] if int8 else x[:1, :16].cpu().numpy()
        assert np.array_equal(kc[0, 2147483644 % slots].cpu().numpy(), want)


# ------------------------------------------------------------------ logits
@pytest.mark.parametrize("vocab,ld,ldo,off", [
    (33, 33, 33, 0), (120007, 120007, 120007, 0), (102401, 102404, 102402, 1), (250001, 250003, 250003, 3),
])
@pytest.mark.parametrize("n_bias", [0, 256, 257, 900])
def test_logits_of_long_bias_lists_and_vocabularies(cuda, vocab, ld, ldo, off, n_bias):
    """Bias lists longer than a block keeps, ids repeated and at the edges of its
    share; vocabularies that take the blocks of a row several turns."""
    torch = cuda
    r = np.random.default_rng(vocab + n_bias)
    rows = 3
    x = (r.normal(size=(rows, ld)) * 4).astype(np.float32)
    edges = np.array([0, 1, vocab - 1, 12799, 12800, 12801, 102399, 102400, 102401, -1, vocab], np.int32)
    lens = np.array([0, 1500, 700])
    hoff = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    hist = np.where(r.random(hoff[-1]) < 0.1, r.choice(edges, hoff[-1]), r.integers(0, vocab, hoff[-1])).astype(np.int32)
    gen = np.array([0, 300, 2200], np.int32)  # the last: nothing generated
    rep = np.array([1.0, 1.7, 0.6], np.float32)
    pres, freq = np.array([0.5, -0.25, 2.0], np.float32), np.array([0.1, 0.3, 0.0], np.float32)
    bids = bvals = boff = None
    if n_bias:
        nbias = np.array([n_bias, n_bias, 0])
        boff = np.concatenate([[0], np.cumsum(nbias)]).astype(np.int32)
        bids = np.where(r.random(boff[-1]) < 0.3, r.choice(edges, boff[-1]), r.integers(0, vocab, boff[-1])).astype(np.int32)
        bvals = r.normal(size=boff[-1]).astype(np.float32)
    keep = r.random((rows, vocab)) < 0.7
    d = [dev(torch, a) for a in (hist, hoff, gen, rep, pres, freq, bids, bvals, boff)]
    mask = dev(torch, nb.pack_mask(keep).view(np.int32))
    buf = torch.zeros(rows * ld + off, device="cuda")
    buf[off:] = dev(torch, x).reshape(-1)
    y = torch.full((rows, ldo), 8.0, device="cuda")
    picks = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    nb.logits_adjust(ptr(buf) + 4 * off, ld, rows, vocab, ptr(y), ldo, *[ptr(t) for t in d], ptr(mask),
                     (vocab + 31) // 32, -1e9, ptr(picks))
    got = y.cpu().numpy()
    want, size = logits_ref(x[:, :vocab], hist, hoff, gen, rep, pres, freq, bids, bvals, boff, keep, -1e9)
    assert np.all(got[:, vocab:] == 8.0)
    # n_bias additions in list order, one rounding each
    assert np.all(np.abs(got[:, :vocab] - want) <= (LOGIT_TOL + n_bias * 2.0 ** -24) * size)
    assert np.array_equal(picks.cpu().numpy(), got[:, :vocab].argmax(1))


# ------------------------------------------------------------------ two threads
def test_two_threads_on_streams_of_their_own(cuda):
    """Every operator from two host threads at once equals the calls of one."""
    torch = cuda
    sets = [all_calls(torch, s) for s in (11, 12)]
    want = []
    for calls, outs, _ in sets:
        for f in calls:
            f(None)
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _, outs, _ in sets:
        for o in outs:
            o.fill_(3)
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            for _ in range(50):
                for f in sets[i][0]:
                    f(streams[i].cuda_stream)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for (_, outs, _), w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(outs, w))


FIRST = """
import sys
sys.path.insert(0, "tests")
import torch
torch.cuda.init()
from test_gpu_draft import all_calls, nb
stream = torch.cuda.Stream()
nb.attend_tree, eager = (lambda *a, **k: None), nb.attend_tree  # all_calls runs it once
calls, outs, hold = all_calls(torch, 3)
nb.attend_tree = eager
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=stream):
    for f in calls:
        f(stream.cuda_stream)
for _ in range(3):
    g.replay()
torch.cuda.synchronize()
got = [o.clone() for o in outs]
for f in calls:
    f(None)
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, outs)), "replay differs"
print("ok")
"""


def test_first_calls_of_a_process_may_be_captured(cuda):
    """No call needs an eager one before it."""
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=os.path.join(ROOT, "tests")))
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-2000:]
