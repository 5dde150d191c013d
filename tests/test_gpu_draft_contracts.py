"""What the header promises of the operators for drafted tokens at the edges of
its wording: rows skipped inside a prompt longer than its ring, and the like.

Tolerances are those of the 64-bit references (Tree.want, ROPE_TOL, LOGIT_TOL)
where nothing else stands beside the comparison.
"""
import numpy as np
import pytest
from conftest import cact_pack, nb, orc
from test_gpu_draft import LOGIT_TOL, ROPE_TOL, Tree, dev, logits_ref, ptr, quant_ref, rope_ref
from test_gpu_kernels import close, make_weight

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ waits that gave up
class _Word:
    """One int32 of device memory as torch takes it."""

    def __init__(self, address):
        self.__cuda_array_interface__ = dict(shape=(1,), typestr="<i4", data=(address, False), version=2)


def test_a_wait_that_gave_up_is_told_once(cuda):
    """The flag the kernels raise, raised here from outside: read, then clear.
    Calls that wait as they should leave it alone."""
    torch = cuda
    Tree(2, 20, 4, 2, 48, 64, 90, 80, True, seed=1).check(torch)
    torch.cuda.synchronize()
    assert not nb.take_wait_error()
    flag = torch.as_tensor(_Word(nb.wait_flag()), device="cuda")
    flag.fill_(1)
    torch.cuda.synchronize()
    Tree(2, 20, 4, 2, 48, 64, 90, 80, True, seed=1).check(torch)  # no call clears or minds it
    torch.cuda.synchronize()
    assert nb.take_wait_error() and not nb.take_wait_error()
    assert int(flag[0]) == 0


def test_the_wait_flag_may_be_copied_in_a_graph(cuda):
    torch = cuda
    flag = torch.as_tensor(_Word(nb.wait_flag()), device="cuda")
    seen = torch.zeros(1, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        seen.copy_(flag)
    for v in (0, 1):
        flag.fill_(v)
        g.replay()
        torch.cuda.synchronize()
        assert int(seen[0]) == v
    assert nb.take_wait_error() and not nb.take_wait_error()


# ------------------------------------------------------------------ the way back of a rotation
SCALINGS = [(None, 1.0), (("linear", 4.0, 0), 1.0), (("by_parts", 32.0, 4096.0), 0.1 * np.log(32.0) + 1.0)]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("scaling,m", SCALINGS)
def test_rope_and_its_inverse_return_x(cuda, inter, scaling, m):
    """Taking a rotation out again: with mscale = 1 / m the rows come back."""
    torch = cuda
    M, heads, dim, rot = 300, 3, 64, 48
    rng = np.random.default_rng(4)
    x = rng.normal(size=(M, heads * dim)).astype(np.float32)
    pos = dev(torch, rng.integers(0, 1 << 20, M).astype(np.int32))
    y = dev(torch, x)
    for inverse in (False, True):
        sc = None
        if scaling is not None:
            sc = nb.RopeScaling(scaling[0], scaling[1], trained=scaling[2], mscale=1.0 / m if inverse else 0.0)
        nb.rope(ptr(y), heads * dim, ptr(y), heads * dim, ptr(pos), M, heads, dim, rot_dim=rot, interleaved=inter,
                scaling=sc, inverse=inverse)
    _, size = rope_ref(x, pos.cpu().numpy(), heads, dim, rot, 10000.0, inter, None, False)
    # With e = ROPE_TOL (|x1| + |x2|): the rotation's errors, at most m e each, are both turned
    # back and divided by m: 2 e. The way back adds its own bound of the rotated pair,
    # ROPE_TOL (|y1| + |y2|) / m, at most sqrt(2) e. 1 / m is rounded once.
    assert np.all(np.abs(y.cpu().numpy() - x) <= (2 + 2 ** 0.5) * ROPE_TOL * size + 2.0 ** -24 * np.abs(x))


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("scaling,m", SCALINGS)
def test_rope_inverse_is_the_transpose(cuda, inter, scaling, m):
    """The gradient's way back: <rope(x), g> = <x, inverse(g)> of every pair, by
    the 64-bit rotation and by differences of it."""
    torch = cuda
    M, heads, dim, rot = 40, 2, 32, 24
    rng = np.random.default_rng(5)
    x, g = (rng.normal(size=(M, heads * dim)) for _ in range(2))
    g = g.astype(np.float32)
    pos = rng.integers(0, 1 << 20, M).astype(np.int32)
    sc = None if scaling is None else nb.RopeScaling(scaling[0], scaling[1], trained=scaling[2])
    gd, pd = dev(torch, g), dev(torch, pos)
    out = torch.zeros(M, heads * dim, device="cuda")
    nb.rope(ptr(gd), heads * dim, ptr(out), heads * dim, ptr(pd), M, heads, dim, rot_dim=rot, interleaved=inter,
            scaling=sc, inverse=True)
    got = out.cpu().numpy()

    def rotated(a):
        return rope_ref(a, pos, heads, dim, rot, 10000.0, inter, scaling, False)[0]

    _, size = rope_ref(g, pos, heads, dim, rot, 10000.0, inter, scaling, False)
    for d in range(dim):  # one value of every head and row at a time; the map is linear
        step = np.zeros((M, heads, dim))
        step[:, :, d] = 0.5
        step = step.reshape(M, -1)
        diff = (rotated(x + step) - rotated(x - step)) * g
        want = diff.reshape(M, heads, dim).sum(-1)
        # the differences' own rounding in 64 bits: below 2^-44 of values below 100
        tol = ROPE_TOL * size.reshape(M, heads, dim)[:, :, d] + 2.0 ** -40
        assert np.all(np.abs(got.reshape(M, heads, dim)[:, :, d] - want) <= tol)


# ------------------------------------------------------------------ prompts longer than their rings
def prompt_rows(rng, sessions, slots, valid, holes, pad):
    """Rows of sessions one after another: `pad` skipped ones, `valid[s]`
    consecutive positions with skipped ones among them, `pad` again."""
    sess, pos = [], []
    for s in range(sessions):
        p = [-1] * pad
        first = int(rng.integers(0, 4 * slots))
        for i in range(valid[s]):
            while rng.random() < holes:
                p.append(-int(rng.integers(1, 1 << 31)))
            p.append(first + i)
        p += [-1] * pad
        sess += [s] * len(p)
        pos += p
    return np.array(sess, np.int32), np.array(pos, np.int32)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("slots,valid,holes,pad", [
    (16, (20,), 0.0, 0), (16, (20,), 0.2, 0),
    (1, (9, 1, 4), 0.5, 2), (3, (50, 3, 2, 17), 0.3, 5), (16, (50, 3, 16, 33, 17), 0.1, 1),
    (70, (300, 71, 140, 2), 0.9, 40), (64, (1000, 65), 0.5, 0), (700, (1900, 1400, 701, 2300), 0.02, 300),
    (500, (600, 1000, 999, 501), 0.0, 424),   # a padded batch
    (2000, (4500,), 0.3, 6000),
])
def test_rows_skipped_inside_a_prompt_longer_than_its_ring(cuda, int8, slots, valid, holes, pad):
    """The ring ends as if the rows had been written one by one: the row of the
    latest position in every slot, its codes with its scale."""
    torch = cuda
    rng = np.random.default_rng(slots + len(valid))
    S, kvh, qk, vh = len(valid), 2, 48, 64
    sess, pos = prompt_rows(rng, S, slots, valid, holes, pad)
    M, ld = len(pos), kvh * (qk + vh)
    x = (rng.normal(size=(M, ld)) * rng.choice([1e-2, 1.0, 30.0], (M, 1))).astype(np.float32)
    k, v = x[:, : kvh * qk].reshape(M, kvh, qk), x[:, kvh * qk:].reshape(M, kvh, vh)
    (ck, sk), (cv, sv) = (quant_ref(k), quant_ref(v)) if int8 else ((k, None), (v, None))
    last = {}
    for i in range(M):
        if pos[i] >= 0:
            last[int(sess[i]), int(pos[i]) % slots] = i
    want = [np.full((S, slots, kvh, d), 5, c.dtype) for d, c in ((qk, ck), (vh, cv))]
    scales = [np.full((S, slots, kvh), 0.5, np.float32) for _ in range(2)]
    for (s, n), i in last.items():
        want[0][s, n], want[1][s, n] = ck[i], cv[i]
        if int8:
            scales[0][s, n], scales[1][s, n] = sk[i], sv[i]
    xd, sd, pd = dev(torch, x), dev(torch, sess), dev(torch, pos)
    for _ in range(4):
        ring = [torch.full((S, slots, kvh, d), 5, dtype=torch.int8 if int8 else torch.float32, device="cuda")
                for d in (qk, vh)]
        sc = [torch.full((S, slots, kvh), 0.5, device="cuda") if int8 else None for _ in range(2)]
        nb.kv_append(ptr(xd), ld, ptr(xd) + 4 * kvh * qk, ld, ptr(sd), ptr(pd), M, int8, S, slots, kvh, qk, vh,
                     ptr(ring[0]), ptr(ring[1]), ptr(sc[0]), ptr(sc[1]))
        for a, w in zip(ring, want):
            assert np.array_equal(a.cpu().numpy(), w)
        if int8:
            for a, w in zip(sc, scales):
                assert np.array_equal(a.cpu().numpy(), w)


# ------------------------------------------------------------------ keys that are not finite
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,heads,kvh,qk,vh", [(1, 4, 2, 48, 64), (2, 12, 2, 48, 64), (5, 4, 2, 128, 128),
                                               (3, 3, 3, 20, 36), (9, 12, 2, 48, 64), (17, 4, 2, 128, 128)])
def test_a_score_of_minus_infinity_weighs_nothing(cuda, int8, T, heads, kvh, qk, vh):
    """A seen key that every query meets with a score of -inf has weight 0: the
    answer is the one without it, in the ring and in the draft, whichever form runs."""
    torch = cuda
    c = Tree(2, T, heads, kvh, qk, vh, 90, 80, int8, seed=T)
    first = c.q[:, :, : heads * qk].reshape(2, T, heads, qk)
    first[..., 5] = np.abs(first[..., 5]) + 0.25       # a view: every query is positive there
    at = [int(c.hi[b, 0] - 7) % 90 for b in range(2)]
    want, tol = c.want()
    for b in range(2):
        c.hi[b], c.lo[b] = c.hi[b], c.hi[b] - 20
    with_it = c.mask.copy()
    c.mask &= ~np.uint32(1)                            # node 0 unseen, and the ring's place left out:
    lo, hi = c.lo.copy(), c.hi.copy()
    seen = c.seen
    c.seen = lambda b, t: ([s for s in seen(b, t)[0] if s != at[b]], seen(b, t)[1])
    want, tol = c.want()
    c.seen, c.mask = seen, with_it
    for b in range(2):
        if int8:
            c.k[b, at[b]] = c.tk[b, 0] = 0
            c.k[b, at[b], :, 5] = c.tk[b, 0, :, 5] = -100
            c.ks[b, at[b]] = c.tks[b, 0] = np.inf
        else:
            c.k[b, at[b], :, 5] = c.tk[b, 0, :, 5] = -np.inf
    got = c.run(torch).cpu().numpy()
    assert np.array_equal(lo, c.lo) and np.array_equal(hi, c.hi)
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / np.maximum(tol, 1e-30)).max())
    # a NaN among the keys a row sees is the row's answer
    if not int8:
        c.k[:, :, :, 5] = np.nan
        assert np.all(np.isnan(c.run(torch).cpu().numpy()))


@pytest.mark.parametrize("int8", [False, True])
def test_keys_at_the_top_of_the_range(cuda, int8):
    """Keys and scales near the largest float under queries small enough for
    finite scores."""
    torch = cuda
    for T in (1, 2, 9):
        c = Tree(2, T, 12, 2, 48, 64, 90, 80, int8, seed=T)
        c.q = np.clip(c.q, -4, 4) * np.float32(2.0 ** -122)
        if int8:
            for s in (c.ks, c.tks):
                s *= np.float32(2.0 ** 121)
        else:
            c.k, c.tk = (np.clip(a, -4, 4) * np.float32(2.0 ** 122) for a in (c.k, c.tk))
            c.k[:, ::7, :, 3] = np.float32(3.4028234663852886e38)
            c.tk[:, :, :, 3] = -np.float32(3.4028234663852886e38)
        c.check(torch)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,heads,kvh,qk,vh,slots", [(3, 12, 2, 48, 64, 90), (20, 12, 2, 48, 64, 90), (9, 16, 2, 128, 128, 200),
                                                     (24, 4, 1, 64, 64, 4200), (2, 6, 1, 48, 64, 9000)])
def test_padding_nodes_with_queries_that_are_no_numbers(cuda, int8, T, heads, kvh, qk, vh, slots):
    """Nodes whose queries hold NaN get NaN, or zeros where they see nothing; the
    others are as they would be without them."""
    torch = cuda
    c = Tree(2, T, heads, kvh, qk, vh, slots, slots - 5, int8, seed=T)
    blind, seeing = T - 1, 1                            # the last sees nothing at all
    c.mask[:, blind] = 0
    c.hi[:, blind] = -1
    want, tol = c.want()
    c.q[:, blind, 3] = c.q[:, seeing, ::7] = np.nan
    got = c.run(torch).cpu().numpy()
    others = [t for t in range(T) if t not in (blind, seeing)]
    assert np.all(np.abs(got - want)[:, others] <= tol[:, others])
    first = (np.arange(0, c.ldq, 7)[:, None] // qk == np.arange(heads)).any(0)   # heads with a NaN
    if blind != seeing:
        assert np.isnan(got[:, seeing][:, first]).all()
    assert np.all(got[:, blind] == 0.0)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T,heads,kvh,qk,vh,slots", [(65, 4, 1, 48, 64, 300), (40, 8, 2, 64, 64, 90), (33, 8, 2, 128, 128, 200),
                                                     (70, 2, 1, 128, 128, 4200), (150, 1, 1, 48, 64, 5000)])
def test_every_row_done_again(cuda, int8, T, heads, kvh, qk, vh, slots):
    """Keys above 2^96 under queries as small: no row of a tile can stay with split
    operands, whole and partial results alike."""
    torch = cuda
    c = Tree(1, T, heads, kvh, qk, vh, slots, slots - 9, int8, seed=T)
    c.q = c.q * np.float32(2.0 ** -110)
    for n in ("ks", "tks") if int8 else ("k", "tk"):
        setattr(c, n, getattr(c, n) * np.float32(2.0 ** 110))
    c.check(torch)


# ------------------------------------------------------------------ the largest counts
MOST = 2 ** 31 - 1


def _pieces(n, step=1 << 27):
    return [slice(i, min(n, i + step)) for i in range(0, n, step)]


def test_rope_of_the_largest_row_count(cuda):
    """2^31 - 1 rows in one call: every row as in calls of some of them."""
    torch = cuda
    x = torch.empty(MOST, 2, device="cuda")
    pos = torch.empty(MOST, dtype=torch.int32, device="cuda")
    for s in _pieces(MOST):
        i = torch.arange(s.start, s.stop, device="cuda")
        x[s, 0], x[s, 1], pos[s] = (i % 1009).float(), (i % 997).float(), (i % 65537).int()
    nb.rope(ptr(x), 2, ptr(x), 2, ptr(pos), MOST, 1, 2)
    torch.cuda.synchronize()
    for s in _pieces(MOST):
        i = torch.arange(s.start, s.stop, device="cuda")
        y = torch.stack([(i % 1009).float(), (i % 997).float()], 1)
        nb.rope(ptr(y), 2, ptr(y), 2, ptr(pos[s]), s.stop - s.start, 1, 2)
        assert torch.equal(y, x[s])
    del x, pos, i, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("int8", [False, True])
def test_append_and_read_of_the_largest_row_count(cuda, int8):
    """2^31 - 1 rows into a ring of as many places, and back."""
    torch = cuda
    src, pos = torch.empty(MOST, device="cuda"), torch.empty(MOST, dtype=torch.int32, device="cuda")
    for s in _pieces(MOST):
        i = torch.arange(s.start, s.stop, device="cuda")
        src[s], pos[s] = (i % 1009 + 1).float(), (MOST - 1 - i).int()
    sess = torch.zeros(MOST, dtype=torch.int32, device="cuda")
    ring = [torch.empty(MOST, dtype=torch.int8 if int8 else torch.float32, device="cuda") for _ in range(2)]
    sc = [torch.empty(MOST, device="cuda") if int8 else None for _ in range(2)]
    nb.kv_append(ptr(src), 1, ptr(src), 1, ptr(sess), ptr(pos), MOST, int8, 1, MOST, 1, 1, 1, ptr(ring[0]),
                 ptr(ring[1]), ptr(sc[0]), ptr(sc[1]))
    back = torch.zeros(MOST, device="cuda")
    for values in (False, True):
        back.zero_()
        nb.kv_read(ptr(ring[0]), ptr(ring[1]), ptr(sc[0]), ptr(sc[1]), int8, 1, MOST, 1, 1, 1, ptr(sess), ptr(pos),
                   MOST, None if values else ptr(back), 1, ptr(back) if values else None, 1)
        for s in _pieces(MOST):
            # int8: the scale is one value's 127th, rounded, and 127 times that rounded again
            want = src[s] / torch.full_like(src[s], 127.0) * 127.0 if int8 else src[s]
            assert torch.equal(back[s], want)
    del src, pos, sess, ring, sc, back, want, i
    torch.cuda.empty_cache()


def test_logits_of_the_largest_row_count(cuda):
    """2^31 - 1 rows of one logit, in place, each with its pick."""
    torch = cuda
    x = torch.empty(MOST, device="cuda")
    for s in _pieces(MOST):
        x[s] = (torch.arange(s.start, s.stop, device="cuda") % 1009).float()
    picks = torch.full((MOST,), -1, dtype=torch.int32, device="cuda")
    nb.logits_adjust(ptr(x), 1, MOST, 1, ptr(x), 1, picks_ptr=ptr(picks))
    for s in _pieces(MOST):
        assert torch.equal(x[s], (torch.arange(s.start, s.stop, device="cuda") % 1009).float())
        assert not picks[s].any()
    del x, picks
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ long sums
@pytest.mark.parametrize("shape", [(1, 4, 1, 128, 128, 5651), (2, 4, 1, 32, 32, 6007), (1, 12, 2, 48, 64, 9001),
                                   (9, 4, 1, 128, 128, 5651), (4, 12, 2, 48, 64, 9001), (16, 12, 2, 64, 64, 7013)])
@pytest.mark.parametrize("int8", [False, True])
def test_long_sums_stay_within_a_quarter_of_the_32_bit_forms_error(cuda, int8, shape):
    """Against 64 bits, relative to the whole output: at most 1.25 times the error
    of the same attention in plain 32-bit products and sums, or 1.5 * 2^-22 where
    that is more. The floor is the kernels' own arithmetic, as independent errors
    of the weights: an exponential's 2^-22 (rms 1.4e-7), the rounding of its argument
    of up to 8 (2^-22 ln 2, rms 1.0e-7), the 22 bits of query, key and weight (below
    0.7e-7 each), the f32 additions of a warp's blocks (at most 90 here, 1.6e-7 as a
    random walk): together 2.7e-7. Sums left to accumulators that truncate were
    at 8.4e-7 over 5651 positions."""
    torch = cuda
    T, heads, kvh, qk, vh, ctx = shape
    c = Tree(1, T, heads, kvh, qk, vh, ctx, ctx, int8, seed=ctx)
    c.lo[:] = 0
    c.hi[:] = ctx - 1
    c.mask[:] = 0
    got = c.run(torch)[0].double()
    k, v = (torch.from_numpy(a[0].astype(np.float64)).cuda() for a in (c.k, c.v))
    if int8:
        k, v = (a * torch.from_numpy(s[0].astype(np.float64)).cuda()[..., None] for a, s in ((k, c.ks), (v, c.vs)))
    q = torch.from_numpy(c.q[0, :, : heads * qk].reshape(T, heads, qk)).cuda().double()

    def attend(dt):
        kk, vv = (a.to(dt).repeat_interleave(heads // kvh, 1).transpose(0, 1) for a in (k, v))
        s = q.to(dt).transpose(0, 1) @ kk.transpose(1, 2) / qk ** 0.5
        w = torch.exp(s - s.amax(-1, keepdim=True))
        return (w @ vv / w.sum(-1, keepdim=True)).transpose(0, 1).double()

    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    want, plain = attend(torch.float64), attend(torch.float32)
    torch.backends.cuda.matmul.allow_tf32 = old
    mine, theirs = (float((x - want).norm() / want.norm()) for x in (got, plain))
    assert mine <= max(1.25 * theirs, 1.5 * 2.0 ** -22), (mine, theirs)


# ------------------------------------------------------------------ a layer as a server runs it
def fake_quantised(torch, q, rows, heads, qk):
    """Queries [rows][heads * qk] through the int8 codes and back, in place: the
    scales of nd_kv_quant, the values of nd_kv_read."""
    codes = torch.empty(rows, heads, qk, dtype=torch.int8, device="cuda")
    scales = torch.empty(rows, heads, device="cuda")
    zero = torch.zeros(rows, dtype=torch.int32, device="cuda")
    nb.kv_quant(ptr(q), rows * heads, qk, ptr(codes), ptr(scales))
    nb.kv_read(ptr(codes), None, ptr(scales), None, True, rows, 1, heads, qk, qk, None, ptr(zero), rows, ptr(q),
               heads * qk, None, 0)


def test_an_int8_draft_is_verified_as_the_reference_decodes(cuda):
    """Queries fake-quantised on the device equal the reference's to the bit, and
    each node of a chain equals the reference's decode step (fake-quantised query,
    the earlier nodes in the ring)."""
    torch = cuda
    B, T, H, kvh, qk, vh, slots = 3, 6, 12, 2, 48, 64, 96
    c = Tree(B, T, H, kvh, qk, vh, slots, 70, True, seed=3, mask="chain")
    q = dev(torch, c.q)
    fake_quantised(torch, q, B * T, H, qk)
    got_q = q.cpu().numpy()
    want_q = np.stack([orc.fake_quant(v) for v in c.q.reshape(-1, qk)]).reshape(c.q.shape)
    assert np.array_equal(got_q, want_q) and not np.array_equal(got_q, c.q)
    c.q = got_q
    got = c.check(torch)
    _, tol = c.want()
    for b in range(B):
        k, v, ks, vs = (a[b].copy() for a in (c.k, c.v, c.ks, c.vs))
        for t in range(T):
            at = int(c.hi[b, t]) + 1 + t
            k[at % slots], v[at % slots], ks[at % slots], vs[at % slots] = c.tk[b, t], c.tv[b, t], c.tks[b, t], c.tvs[b, t]
            want = orc.attend_step(got_q[b, t], slots, int(c.lo[b, t]), at, H, kvh, qk, vh, kq=k.ravel(),
                                   ks=ks.ravel(), vq=v.ravel(), vs=vs.ravel())
            # the oracle sums in f32 itself: within its own rounding, the bound again
            assert np.all(np.abs(got[b, t] - np.asarray(want).reshape(H, vh)) <= 2 * tol[b, t])


@pytest.mark.parametrize("int8", [False, True])
def test_a_drafted_layer_from_projection_to_picks(cuda, int8):
    """Hidden states to picks of a tree's nodes as one run of calls: project q | k
    | v, rotate, append to the draft, attend, project to logits, correct and pick,
    append the accepted path. Every step's output is held against its reference
    on what the step before it left."""
    torch = cuda
    B, H, kvh, qk, vh, slots, V, d = 3, 12, 2, 48, 64, 90, 812, 768
    parents, path = [-1, 0, 0, 1, 3, 2, 4], [0, 1, 3, 4, 6]
    T, N = len(parents), 3 * len(parents)
    depth = [0] * T
    for t, p in enumerate(parents):
        depth[t] = depth[p] + 1 if p >= 0 else 0
    rng = np.random.default_rng(8)
    cb = cact_pack.random_codebook(np.random.default_rng(9))
    levels = cact_pack.codebook_levels(cb, 2)
    shapes = (H * qk, kvh * qk, kvh * vh)
    mats = [make_weight(torch, o, d, 2, 50 + i, cb) for i, o in enumerate(shapes)]
    head = make_weight(torch, V, d, 2, 60, cb)
    ld = sum(shapes)
    c = Tree(B, T, H, kvh, qk, vh, slots, 80, int8, seed=12)
    c.mask = np.repeat(nb.tree_mask(parents)[None], B, 0)
    ring = [dev(torch, a) for a in (c.k, c.v, c.ks, c.vs)]
    pos = np.array([[c.hi[b, 0] + 1 + depth[t] for t in range(T)] for b in range(B)], np.int32).ravel()
    sess, node = np.repeat(np.arange(B), T).astype(np.int32), np.tile(np.arange(T), B).astype(np.int32)
    kept = np.where(np.isin(node, path), pos, -1).astype(np.int32)
    posd, sessd, noded, keptd, lo, hi, mask = (dev(torch, a) for a in (pos, sess, node, kept, c.lo, c.hi, c.mask.view(np.int32)))
    hist = rng.integers(0, V, 40 * N).astype(np.int32)
    off = (np.arange(N + 1) * 40).astype(np.int32)
    gen = off[:-1] + 20
    rep, pres, freq = (rng.uniform(a, b, N).astype(np.float32) for a, b in ((1.0, 1.5), (0.0, 0.5), (0.0, 0.3)))
    keep = rng.random((N, V)) < 0.5
    hd, od, gd, rd, pd, fd, bits = (dev(torch, a) for a in (hist, off, gen, rep, pres, freq, nb.pack_mask(keep).view(np.int32)))
    dt = torch.int8 if int8 else torch.float32
    draft = [torch.zeros(B, T, kvh, w, dtype=dt, device="cuda") for w in (qk, vh)]
    draft += [torch.zeros(B, T, kvh, device="cuda") if int8 else None for _ in range(2)]
    x = (rng.normal(size=(N, d)) * 3).astype(np.float32)
    xd, xh, oh = dev(torch, x), torch.zeros(N, d, device="cuda"), torch.zeros(N, d, device="cuda")
    rows, q = torch.zeros(N, ld, device="cuda"), torch.zeros(N, H * qk, device="cuda")
    out, logits = torch.zeros(B, T, H, vh, device="cuda"), torch.zeros(N, V, device="cuda")
    picks = torch.zeros(N, dtype=torch.int32, device="cuda")
    at_k, at_v = 4 * H * qk, 4 * (H + kvh) * qk

    # ---- the run of calls
    nb.cq_prepare(ptr(xd), N, d, ptr(xh), d)
    nb.cq_project_grouped([(m[1], m[2], o) for m, o in zip(mats, shapes)], d, 2, levels, ptr(xh), d, N, ptr(rows), ld)
    projected = rows.clone()
    nb.rope(ptr(rows), ld, ptr(q), H * qk, ptr(posd), N, H, qk)
    nb.rope(ptr(rows) + at_k, ld, ptr(rows) + at_k, ld, ptr(posd), N, kvh, qk)
    rotated = q.clone()
    if int8:
        fake_quantised(torch, q, N, H, qk)
    nb.kv_append(ptr(rows) + at_k, ld, ptr(rows) + at_v, ld, ptr(sessd), ptr(noded), N, int8, B, T, kvh, qk, vh,
                 *[ptr(a) for a in draft])
    nb.attend_tree(ptr(q), H * qk, *[ptr(a) for a in ring], int8, slots, ptr(lo), ptr(hi), *[ptr(a) for a in draft],
                   ptr(mask), B, T, H, kvh, qk, vh, ptr(out))
    nb.cq_prepare(ptr(out), N, d, ptr(oh), d)
    nb.cq_project(head[1], head[2], V, d, 2, levels, ptr(oh), d, N, ptr(logits), V)
    plain = logits.clone()
    nb.logits_adjust(ptr(logits), V, N, V, ptr(logits), V, ptr(hd), ptr(od), ptr(gd), ptr(rd), ptr(pd), ptr(fd),
                     mask_ptr=ptr(bits), mask_ld=(V + 31) // 32, masked=-1e9, picks_ptr=ptr(picks))
    nb.kv_append(ptr(rows) + at_k, ld, ptr(rows) + at_v, ld, ptr(sessd), ptr(keptd), N, int8, B, slots, kvh, qk, vh,
                 *[ptr(a) for a in ring])

    # ---- each step against its reference
    xh_want = np.stack([mats[0][3].prepare(r) for r in x])
    assert close(projected.cpu().numpy(), np.concatenate([m[3].matmul_prepared(xh_want) for m in mats], 1))
    proj = projected.cpu().numpy()
    for got, a, n in ((rotated, 0, H), (rows[:, H * qk: (H + kvh) * qk], H * qk, kvh)):
        want, size = rope_ref(proj[:, a: a + n * qk], pos, n, qk, qk, 10000.0, False, None, False)
        assert np.all(np.abs(got.cpu().numpy() - want) <= ROPE_TOL * size)
    if int8:
        want = np.stack([orc.fake_quant(v) for v in rotated.cpu().numpy().reshape(-1, qk)])
        assert np.array_equal(q.cpu().numpy().reshape(-1, qk), want)
    r = rows.cpu().numpy()
    k, v = r[:, H * qk: (H + kvh) * qk].reshape(N, kvh, qk), r[:, (H + kvh) * qk:].reshape(N, kvh, vh)
    (ck, sk), (cv, sv) = (quant_ref(k), quant_ref(v)) if int8 else ((k, None), (v, None))
    for a, w in zip(draft, (ck, cv, sk, sv)):
        assert a is None or np.array_equal(a.cpu().numpy().reshape(w.shape), w)
    c.q, c.ldq = q.cpu().numpy().reshape(B, T, H * qk), H * qk
    c.tk, c.tv, c.tks, c.tvs = (None if a is None else a.cpu().numpy() for a in draft)
    want, tol = c.want()
    assert np.all(np.abs(out.cpu().numpy() - want) <= tol)
    o = out.cpu().numpy().reshape(N, d)
    assert close(plain.cpu().numpy(), head[3].matmul_prepared(np.stack([head[3].prepare(a) for a in o])))
    got = logits.cpu().numpy()
    want, size = logits_ref(plain.cpu().numpy(), hist, off, gen, rep, pres, freq, None, None, None, keep, -1e9)
    assert np.all(np.abs(got - want) <= LOGIT_TOL * size)
    assert np.array_equal(picks.cpu().numpy(), got.argmax(1))
    final = [None if a is None else a.copy() for a in (c.k, c.v, c.ks, c.vs)]
    for i in np.flatnonzero(kept >= 0):
        for a, w in zip(final, (ck, cv, sk, sv)):
            if a is not None:
                a[sess[i], kept[i] % slots] = w[i]
    for a, w in zip(ring, final):
        assert a is None or np.array_equal(a.cpu().numpy(), w)


# ------------------------------------------------------------------ the ends of the documented ranges
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("shape", [
    # B, T, heads, kv_heads, qk, vh, slots, ctx
    (1, 3, 301, 1, 48, 64, 40, 33),      # hundreds of query heads a KV head
    (2, 1, 512, 512, 16, 16, 30, 21),    # the most KV heads
    (1, 2, 1024, 512, 4, 4, 20, 17),
    (3, 5, 6, 2, 4, 4, 33, 30),          # the narrowest heads
    (1, 40, 4, 2, 4, 128, 50, 41),
    (2, 20, 2, 1, 128, 16, 7, 7),
])
def test_tree_attention_at_the_ends_of_its_ranges(cuda, int8, shape):
    B, T, heads, kvh, qk, vh, slots, ctx = shape
    Tree(B, T, heads, kvh, qk, vh, slots, ctx, int8, seed=sum(shape), extra=T % 3).check(cuda)


@pytest.mark.parametrize("int8", [False, True])
def test_the_most_nodes(cuda, int8):
    """4096 nodes: 128 mask words a node, a chain and a tree; a few rows by 64 bits."""
    torch = cuda
    for mask in ("chain", "tree"):
        c = Tree(1, 4096, 2, 1, 16, 16, 50, 41, int8, seed=6, mask=mask)
        got = c.run(torch).cpu().numpy()
        rows = sorted({0, 1, 31, 32, 63, 64, 127, 128, 2047, 2048, 4094, 4095})
        seen = {t: c.seen(0, t) for t in rows}
        q, c.T = c.q, 1                 # Tree.want of one node at a time
        for t in rows:
            c.q, c.seen = q[:, t: t + 1], lambda b, u, t=t: seen[t]
            want, tol = c.want()
            assert np.all(np.abs(got[:, t] - want[:, 0]) <= tol[:, 0]), (mask, t)
        assert np.isfinite(got).all()


@pytest.mark.parametrize("T", [1, 3, 20])
def test_a_ring_of_2_to_the_30_places(cuda, T):
    """Windows at both ends of the largest ring, in one call and one row tile."""
    torch = cuda
    slots, d = 1 << 30, 16
    k, v = (torch.zeros(slots, d, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(slots, device="cuda") for _ in range(2))
    near, far = slice(5, 105), slice(slots - 100, slots)
    for s in (near, far):
        v[s] = torch.randint(-127, 128, (100, d), dtype=torch.int8, device="cuda")
    q = torch.zeros(T, d, device="cuda")
    lo = torch.tensor([5 if t % 2 else slots - 100 for t in range(T)], dtype=torch.int32, device="cuda")
    hi = lo + 99
    if T > 2:  # across the ring's end: the last 100 places and the first 105
        lo[2], hi[2] = slots - 100, slots + 104
    out = torch.zeros(T, d, device="cuda")
    nb.attend_tree(ptr(q), d, ptr(k), ptr(v), ptr(ks), ptr(vs), True, slots, ptr(lo), ptr(hi), None, None, None, None,
                   None, 1, T, 1, 1, d, d, ptr(out))
    want = [(v[near] if t % 2 else v[far]).double().mean(0) for t in range(T)]
    if T > 2:
        want[2] = torch.cat([v[far], v[:105]]).double().mean(0)
    # weights of 1: sums of whole numbers below 2^24, one division
    assert ((out.double() - torch.stack(want)).abs() <= 2.0 ** -20 * 127).all()
    del k, v, ks, vs
    torch.cuda.empty_cache()


def test_append_of_the_most_heads(cuda):
    torch = cuda
    for int8 in (False, True):
        M, kvh, qk, vh = 5, 512, 12, 256
        x = np.random.default_rng(0).normal(size=(M, kvh * (qk + vh))).astype(np.float32)
        xd = dev(torch, x)
        pos = torch.arange(M, dtype=torch.int32, device="cuda") % 2
        sess = torch.arange(M, dtype=torch.int32, device="cuda") // 2
        dt = torch.int8 if int8 else torch.float32
        ring = [torch.zeros(3, 2, kvh, w, dtype=dt, device="cuda") for w in (qk, vh)]
        sc = [torch.zeros(3, 2, kvh, device="cuda") if int8 else None for _ in range(2)]
        nb.kv_append(ptr(xd), x.shape[1], ptr(xd) + 4 * kvh * qk, x.shape[1], ptr(sess), ptr(pos), M, int8, 3, 2, kvh,
                     qk, vh, ptr(ring[0]), ptr(ring[1]), ptr(sc[0]), ptr(sc[1]))
        for a, s, part, w in ((ring[0], sc[0], x[:, : kvh * qk], qk), (ring[1], sc[1], x[:, kvh * qk:], vh)):
            want = part.reshape(M, kvh, w)
            if int8:
                want, scales = quant_ref(want)
                assert np.array_equal(s.cpu().numpy().reshape(6, kvh)[:M], scales)
            assert np.array_equal(a.cpu().numpy().reshape(6, kvh, w)[:M], want)


def test_logits_of_the_largest_vocabulary(cuda):
    """2^30 ids: history, biases and mask at both ends, in place."""
    torch = cuda
    V = 1 << 30
    x = torch.zeros(V, device="cuda")
    x[V - 2], x[3], x[V // 2] = 9.0, 8.0, 8.5
    mask = torch.full((V // 32,), -1, dtype=torch.int32, device="cuda")
    mask[V // 64] = -2                                  # V / 2 forbidden
    hist = torch.tensor([V - 2, V - 1, V - 2, -1], dtype=torch.int32, device="cuda")
    ids = torch.tensor([V - 1, 0, V - 1], dtype=torch.int32, device="cuda")
    vals = torch.tensor([2.0, 1.0, 4.0], device="cuda")
    ends = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (4, 3)]
    rep, pres, freq = (torch.tensor([a], device="cuda") for a in (2.0, 0.25, 0.5))
    picks = torch.zeros(1, dtype=torch.int32, device="cuda")
    nb.logits_adjust(ptr(x), V, 1, V, ptr(x), V, ptr(hist), ptr(ends[0]), None, ptr(rep), ptr(pres), ptr(freq), ptr(ids),
                     ptr(vals), ptr(ends[1]), ptr(mask), V // 32, -1e9, ptr(picks))
    at = [V - 2, V - 1, V // 2, 3, 0]
    assert x[at].cpu().tolist() == [9.0 / 2 - 1.25, 6.0 - 0.75, -1e9, 8.0, 1.0] and int(picks[0]) == 3
    x[at] = 0.0
    assert not x.any()
    del x, mask
    torch.cuda.empty_cache()


@pytest.mark.parametrize("int8", [False, True])
def test_a_joined_decode_step_in_two_graphs(cuda, int8):
    """One token over a long ring (partial results in scratch, a second kernel):
    two graphs replayed on two streams at once, and again."""
    torch = cuda
    sets = []
    for seed in (1, 2):
        c = Tree(1, 1, 6, 1, 48, 64, 9000, 8900, int8, seed=seed, drafted=False)
        want = torch.from_numpy(c.check(torch)).cuda()
        out, stream, g = torch.zeros_like(want), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            c.call(c.keep, out, stream.cuda_stream)
        sets.append((c, want, out, stream, g))
    for _ in range(5):
        for _, _, out, _, _ in sets:
            out.fill_(3)
        torch.cuda.synchronize()
        for _, _, _, stream, g in sets:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, want, out, _, _ in sets)
