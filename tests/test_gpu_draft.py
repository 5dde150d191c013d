"""GPU parity of the operators for drafted tokens (nd_rope, nd_kv_append,
nd_kv_read, nd_attend_tree, nd_logits_adjust) against plain 64-bit forms.

Tolerances come from the arithmetic, beside each comparison: an f32 rounding
is off by at most 2^-24 of the value, an f16 high part with its remainder by
2^-22, a tensor-core accumulation truncates by at most 2^-23 of the running
sum per step.
"""
import ctypes as C
import importlib.util
import os

import numpy as np
import pytest
from conftest import ROOT, nb, orc

pytestmark = pytest.mark.gpu


def dev(torch, a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------ rope
def rope_ref(x, pos, heads, dim, rot, theta, inter, scaling, inverse):
    """x [M][heads * dim] in 64 bits."""
    M = len(pos)
    y = x.astype(np.float64).reshape(M, heads, dim).copy()
    j = np.arange(rot // 2)
    w = theta ** (-2.0 * j / rot)
    m = 1.0
    if scaling is not None:
        kind, factor, trained = scaling
        if kind == "linear":
            w = w / factor
        else:
            keep = np.clip((trained * w / (2 * np.pi) - 1.0) / 31.0, 0.0, 1.0)
            w = w * keep + w / factor * (1 - keep)
            m = 0.1 * np.log(factor) + 1.0
    a = pos.astype(np.float64)[:, None] * w
    c, s = (m * np.cos(a))[:, None], (m * np.sin(a))[:, None] * (-1 if inverse else 1)
    i0, i1 = (2 * j, 2 * j + 1) if inter else (j, j + rot // 2)
    x0, x1 = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    size = np.zeros_like(y)
    size[..., i0] = size[..., i1] = m * (np.abs(x0) + np.abs(x1))
    return y.reshape(M, -1), size.reshape(M, -1)


# Per rotated value: the reduced turn is rounded once to f32 (2^-26 turns =
# 9.4e-8 rad), sine and cosine are off by 2 ulp (1.2e-7), their factor, the two
# products and the sum by 2^-24 each: together below 4.2e-7 of m (|x1| + |x2|).
ROPE_TOL = 4.2e-7


@pytest.mark.parametrize("M,heads,dim,rot,ldx,ldy,off", [
    (1, 1, 2, 2, 2, 2, 0),
    (5, 14, 48, 48, 800, 672, 0),       # the shipped geometry's q|k columns of a projection row
    (700, 3, 64, 32, 192, 200, 0),      # more than one token a block, part of the head
    (3, 2, 128, 128, 256, 256, 0),
    (33, 5, 20, 12, 103, 101, 1),       # odd strides and an odd start: one pair at a time
    (9, 2, 256, 256, 512, 512, 0),
    (2500, 1, 6, 4, 6, 6, 0),
])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("scaling", [None, ("linear", 4.0, 0), ("by_parts", 32.0, 4096.0)])
def test_rope_matches_64_bits(cuda, M, heads, dim, rot, ldx, ldy, off, inter, scaling):
    torch = cuda
    rng = np.random.default_rng(M + heads)
    x = rng.normal(size=(M, ldx)).astype(np.float32)
    pos = rng.integers(0, 1 << 20, M).astype(np.int32)
    pos[0] = 0
    buf = torch.zeros(M * ldx + off, device="cuda")
    buf[off:] = dev(torch, x).reshape(-1)
    y = torch.full((M * ldy + off,), 7.0, device="cuda")
    p = dev(torch, pos)
    sc = None if scaling is None else nb.RopeScaling(scaling[0], scaling[1], trained=scaling[2])
    nb.rope(buf.data_ptr() + 4 * off, ldx, y.data_ptr() + 4 * off, ldy, p.data_ptr(), M, heads, dim, rot_dim=rot,
            theta=500000.0, interleaved=inter, scaling=sc)
    got = y[off:].cpu().numpy().reshape(M, ldy)
    n = heads * dim
    want, size = rope_ref(x[:, :n], pos, heads, dim, rot, 500000.0, inter, scaling, False)
    assert np.all(got[:, n:] == 7.0)  # nothing past the row
    assert np.all(np.abs(got[:, :n] - want) <= ROPE_TOL * size)
    # in place, and back: x returns to itself within two rotations' error
    nb.rope(buf.data_ptr() + 4 * off, ldx, buf.data_ptr() + 4 * off, ldx, p.data_ptr(), M, heads, dim, rot_dim=rot,
            theta=500000.0, interleaved=inter, scaling=sc)
    assert np.array_equal(buf[off:].cpu().numpy().reshape(M, ldx)[:, :n], got[:, :n])
    assert np.array_equal(buf[off:].cpu().numpy().reshape(M, ldx)[:, n:], x[:, n:])
    nb.rope(buf.data_ptr() + 4 * off, ldx, buf.data_ptr() + 4 * off, ldx, p.data_ptr(), M, heads, dim, rot_dim=rot,
            theta=500000.0, interleaved=inter, scaling=sc, inverse=True)
    back = buf[off:].cpu().numpy().reshape(M, ldx)[:, :n]
    want, size = rope_ref(got[:, :n], pos, heads, dim, rot, 500000.0, inter, scaling, True)
    assert np.all(np.abs(back - want) <= ROPE_TOL * size)


def test_rope_leaves_rows_of_negative_position(cuda):
    torch = cuda
    x = torch.randn(6, 96, device="cuda")
    y = torch.full((6, 96), 3.0, device="cuda")
    pos = torch.tensor([4, -1, 9, -7, 0, -2147483648], dtype=torch.int32, device="cuda")
    nb.rope(x.data_ptr(), 96, y.data_ptr(), 96, pos.data_ptr(), 6, 2, 48, rot_dim=24)
    assert torch.all(y[[1, 3, 5]] == 3.0) and torch.equal(y[4], x[4])
    z = x.clone()
    nb.rope(z.data_ptr(), 96, z.data_ptr(), 96, pos.data_ptr(), 6, 2, 48, rot_dim=24)
    assert torch.equal(z[[1, 3, 5]], x[[1, 3, 5]]) and torch.equal(z[[0, 2, 4]], y[[0, 2, 4]])


# ------------------------------------------------------------------ cache rows
def quant_ref(x):
    """quant_into (cache.rs:100-106) in f32 steps."""
    am = np.abs(x).max(-1, keepdims=True).astype(np.float32)
    scale = np.where(am > 0, am / np.float32(127.0), np.float32(1.0)).astype(np.float32)
    y = (x * (np.float32(1.0) / scale)).astype(np.float32)
    r = np.trunc(y)
    r = np.where(np.abs(y - r) >= 0.5, r + np.sign(y), r)
    return np.clip(r, -128, 127).astype(np.int8), scale[..., 0]


RINGS = [
    # M, sessions, slots, kv_heads, qk, vh, extra row floats, start of the buffer
    (1, 1, 1, 1, 16, 32, 0, 0),
    (37, 5, 9, 2, 48, 64, 16, 0),
    (300, 3, 128, 3, 64, 32, 5, 0),    # odd strides: value by value
    (50, 4, 20, 2, 80, 128, 0, 0),
    (50, 4, 20, 1, 7, 9, 0, 3),        # odd widths
    (20, 2, 16, 2, 132, 256, 4, 0),
    (11, 11, 4, 8, 255, 130, 1, 0),
]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("M,S,slots,kvh,qk,vh,extra,off", RINGS)
def test_append_and_read_back(cuda, int8, M, S, slots, kvh, qk, vh, extra, off):
    """Every place a row names holds its values (int8: the reference quantiser's
    codes and scales, bit for bit), every other place what it held before; the
    read gives code * scale."""
    torch = cuda
    rng = np.random.default_rng(M * 7 + qk)
    ld = kvh * (qk + vh) + extra
    x = (rng.normal(size=(M, ld)) * rng.choice([1e-3, 1.0, 50.0], (M, 1))).astype(np.float32)
    x[rng.integers(0, M)] = 0.0
    # distinct places, any order, positions several turns into the ring
    place = rng.permutation(S * slots)[:M]
    M = len(place)
    x = x[:M]
    sess = (place // slots).astype(np.int32)
    pos = (place % slots + slots * rng.integers(0, 5, M)).astype(np.int32)
    skip = rng.random(M) < 0.2
    pos[skip] = -1
    sess[skip & (rng.random(M) < 0.5)] = S + 3
    if M > 2:
        sess[0], pos[0], skip[0] = -1, 1, True
    dt = torch.int8 if int8 else torch.float32
    kc = torch.full((S, slots, kvh, qk), 5, dtype=dt, device="cuda")
    vc = torch.full((S, slots, kvh, vh), 6, dtype=dt, device="cuda")
    ks, vs = (torch.full((S, slots, kvh), 0.5, device="cuda") for _ in range(2)) if int8 else (None, None)
    buf = torch.zeros(M * ld + off, device="cuda")
    buf[off:] = dev(torch, x).reshape(-1)
    base = buf.data_ptr() + 4 * off
    sd, pd = dev(torch, sess), dev(torch, pos)
    nb.kv_append(base, ld, base + 4 * kvh * qk, ld, sd.data_ptr(), pd.data_ptr(), M, int8, S, slots, kvh, qk, vh,
                 ptr(kc), ptr(vc), ptr(ks), ptr(vs))
    k, v = x[:, : kvh * qk].reshape(M, kvh, qk), x[:, kvh * qk: kvh * (qk + vh)].reshape(M, kvh, vh)
    wk, wv = np.full((S, slots, kvh, qk), 5, np.float32), np.full((S, slots, kvh, vh), 6, np.float32)
    if int8:
        wks, wvs = np.full((S, slots, kvh), 0.5, np.float32), np.full((S, slots, kvh), 0.5, np.float32)
        (k, ksc), (v, vsc) = quant_ref(k), quant_ref(v)
    for i in range(M):
        if skip[i]:
            continue
        s, n = sess[i], pos[i] % slots
        wk[s, n], wv[s, n] = k[i], v[i]
        if int8:
            wks[s, n], wvs[s, n] = ksc[i], vsc[i]
    assert np.array_equal(kc.cpu().numpy().astype(np.float32), wk)
    assert np.array_equal(vc.cpu().numpy().astype(np.float32), wv)
    if int8:
        assert np.array_equal(ks.cpu().numpy(), wks) and np.array_equal(vs.cpu().numpy(), wvs)
        wk, wv = wk * wks[..., None], wv * wvs[..., None]
    # read back, into strided rows; skipped rows stay
    lk, lv = kvh * qk + extra, kvh * vh + 2 * extra
    ko, vo = torch.full((M, lk), 9.0, device="cuda"), torch.full((M, lv), 9.0, device="cuda")
    args = (ptr(kc), ptr(vc), ptr(ks), ptr(vs), int8, S, slots, kvh, qk, vh, sd.data_ptr(), pd.data_ptr(), M)
    nb.kv_read(*args, ko.data_ptr(), lk, vo.data_ptr(), lv)
    kw, vw = np.full((M, lk), 9.0, np.float32), np.full((M, lv), 9.0, np.float32)
    for i in range(M):
        if not skip[i]:
            kw[i, : kvh * qk] = wk[sess[i], pos[i] % slots].reshape(-1)
            vw[i, : kvh * vh] = wv[sess[i], pos[i] % slots].reshape(-1)
    assert np.array_equal(ko.cpu().numpy(), kw) and np.array_equal(vo.cpu().numpy(), vw)
    # keys alone, values alone
    k1, v1 = torch.full((M, lk), 9.0, device="cuda"), torch.full((M, lv), 9.0, device="cuda")
    nb.kv_read(*args, k1.data_ptr(), lk, None, 0)
    nb.kv_read(*args, None, 0, v1.data_ptr(), lv)
    assert torch.equal(k1, ko) and torch.equal(v1, vo)


def test_append_equals_the_standalone_quantiser(cuda):
    torch = cuda
    x = torch.randn(40, 2 * 48 + 2 * 64, device="cuda") * 3
    S, kvh = 40, 2
    kc, vc = (torch.zeros(S, 3, kvh, d, dtype=torch.int8, device="cuda") for d in (48, 64))
    ks, vs = (torch.zeros(S, 3, kvh, device="cuda") for _ in range(2))
    pos = torch.arange(40, dtype=torch.int32, device="cuda")
    nb.kv_append(x.data_ptr(), 224, x.data_ptr() + 4 * 96, 224, None, pos.data_ptr(), 40, True, S, 3, kvh, 48, 64,
                 ptr(kc), ptr(vc), ptr(ks), ptr(vs))
    k = x[:, :96].reshape(80, 48).contiguous()
    q, sc = torch.zeros(80, 48, dtype=torch.int8, device="cuda"), torch.zeros(80, device="cuda")
    nb.kv_quant(k.data_ptr(), 80, 48, q.data_ptr(), sc.data_ptr())
    i = torch.arange(40, device="cuda")
    assert torch.equal(kc[i, i % 3].reshape(80, 48), q) and torch.equal(ks[i, i % 3].reshape(-1), sc)


@pytest.mark.parametrize("int8", [False, True])
def test_a_prompt_longer_than_its_ring_keeps_its_last_positions(cuda, int8):
    torch = cuda
    slots, kvh, qk, vh = 16, 2, 48, 64
    lens, first = [50, 3, 16, 33], [0, 100, 7, 5]
    M, S = sum(lens), len(lens)
    x = torch.randn(M, kvh * (qk + vh), device="cuda")
    sess = torch.tensor(np.repeat(np.arange(S), lens), dtype=torch.int32, device="cuda")
    pos = torch.tensor(np.concatenate([f + np.arange(n) for f, n in zip(first, lens)]), dtype=torch.int32,
                       device="cuda")
    ld = kvh * (qk + vh)
    k, v = torch.zeros(M, kvh * qk, device="cuda"), torch.zeros(M, kvh * vh, device="cuda")
    dt = torch.int8 if int8 else torch.float32
    kc, vc = (torch.zeros(S, slots, kvh, d, dtype=dt, device="cuda") for d in (qk, vh))
    ks, vs = (torch.zeros(S, slots, kvh, device="cuda") for _ in range(2)) if int8 else (None, None)
    for _ in range(3):
        nb.kv_append(x.data_ptr(), ld, x.data_ptr() + 4 * kvh * qk, ld, ptr(sess), ptr(pos), M, int8, S, slots, kvh,
                     qk, vh, ptr(kc), ptr(vc), ptr(ks), ptr(vs))
    nb.kv_read(ptr(kc), ptr(vc), ptr(ks), ptr(vs), int8, S, slots, kvh, qk, vh, ptr(sess), ptr(pos), M, ptr(k),
               kvh * qk, ptr(v), kvh * vh)
    i = 0
    for n in lens:
        for p in range(n):
            want = x[i + (p if p >= n - slots else p + (n - 1 - p) // slots * slots)]  # the last row of that slot
            wk, wv = want[: kvh * qk].reshape(kvh, qk), want[kvh * qk:].reshape(kvh, vh)
            if int8:
                (ck, sk), (cv, sv) = quant_ref(wk.cpu().numpy()), quant_ref(wv.cpu().numpy())
                wk, wv = dev(torch, ck * sk[:, None]), dev(torch, cv * sv[:, None])
            assert torch.equal(k[i + p], wk.reshape(-1)) and torch.equal(v[i + p], wv.reshape(-1))
        i += n


def test_append_and_read_past_32_bit_offsets(cuda):
    """A ring of more than 2^31 bytes and values: its last rows."""
    torch = cuda
    S, slots, kvh, qk, vh = 3, 1 << 22, 2, 128, 128  # 3.2e9 int8 codes each
    kc, vc = (torch.zeros(S, slots, kvh, qk, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(S, slots, kvh, device="cuda") for _ in range(2))
    x = torch.randn(4, kvh * (qk + vh), device="cuda")
    sess = torch.tensor([2, 2, 0, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([slots - 1, 3 * slots - 2, slots - 1, 0], dtype=torch.int32, device="cuda")
    ld = kvh * (qk + vh)
    nb.kv_append(x.data_ptr(), ld, x.data_ptr() + 4 * kvh * qk, ld, ptr(sess), ptr(pos), 4, True, S, slots, kvh, qk, vh,
                 ptr(kc), ptr(vc), ptr(ks), ptr(vs))
    ck, sk = quant_ref(x[:, : kvh * qk].reshape(4, kvh, qk).cpu().numpy())
    for i in range(4):
        at = int(pos[i]) % slots
        assert np.array_equal(kc[int(sess[i]), at].cpu().numpy(), ck[i])
        assert np.array_equal(ks[int(sess[i]), at].cpu().numpy(), sk[i])
    k, v = torch.zeros(4, kvh * qk, device="cuda"), torch.zeros(4, kvh * vh, device="cuda")
    nb.kv_read(ptr(kc), ptr(vc), ptr(ks), ptr(vs), True, S, slots, kvh, qk, vh, ptr(sess), ptr(pos), 4, ptr(k),
               kvh * qk, ptr(v), kvh * vh)
    assert np.array_equal(k.cpu().numpy(), (ck * sk[..., None]).reshape(4, -1))
    # and the attention reads the same place: one visible position returns its value
    q = torch.randn(3, 2, qk, device="cuda")
    lo = torch.tensor([slots - 1, 0, 3 * slots - 2], dtype=torch.int32, device="cuda")
    out = torch.zeros(3, 2, vh, device="cuda")
    nb.attend_tree(ptr(q), 2 * qk, ptr(kc), ptr(vc), ptr(ks), ptr(vs), True, slots, ptr(lo), ptr(lo), None, None, None,
                   None, None, 3, 1, 2, kvh, qk, vh, ptr(out))
    cv, sv = quant_ref(x[:, kvh * qk:].reshape(4, kvh, vh).cpu().numpy())
    want = cv * sv[..., None]
    for b, i in ((0, 2), (1, 3), (2, 1)):
        assert np.abs(out[b].cpu().numpy() - want[i]).max() <= 4 * 2.0 ** -23 * np.abs(want[i]).max()


# ------------------------------------------------------------------ tree attention
class Tree:
    """Random inputs of one call, on the host, and their 64-bit answer."""

    def __init__(self, B, T, heads, kvh, qk, vh, slots, ctx, int8, seed, drafted=True, mask="tree", qgain=1.0,
                 vgain=1.0, extra=0):
        r = np.random.default_rng(seed)
        self.__dict__.update(B=B, T=T, heads=heads, kvh=kvh, qk=qk, vh=vh, slots=slots, int8=int8)
        self.ldq = heads * qk + extra
        self.q = (r.normal(size=(B, T, self.ldq)) * qgain).astype(np.float32)
        mk = lambda n, d: r.normal(size=(B, n, kvh, d)).astype(np.float32)  # noqa: E731
        self.k, self.v = mk(slots, qk), mk(slots, vh) * np.float32(vgain)
        self.tk, self.tv = (mk(T, qk), mk(T, vh) * np.float32(vgain)) if drafted else (None, None)
        self.ks = self.vs = self.tks = self.tvs = None
        if int8:
            (self.k, self.ks), (self.v, self.vs) = quant_ref(self.k), quant_ref(self.v)
            if drafted:
                (self.tk, self.tks), (self.tv, self.tvs) = quant_ref(self.tk), quant_ref(self.tv)
        last = r.integers(ctx, ctx + 3 * slots, size=(B, 1)) if ctx else np.full((B, 1), -1)
        n = r.integers(max(1, ctx // 2), ctx + 1, size=(B, 1)) if ctx else 0
        self.hi = np.repeat(last, T, 1).astype(np.int32)
        self.lo = np.repeat(last - n + 1, T, 1).astype(np.int32)
        if not drafted or mask == "chain":
            self.mask = None
        else:
            self.mask = np.stack([nb.tree_mask([-1 if t == 0 else int(r.integers(-1, t)) for t in range(T)])
                                  for _ in range(B)])

    def seen(self, b, t):
        """Ring slots and draft nodes node (b, t) sees."""
        lo, hi = max(int(self.lo[b, t]), 0), int(self.hi[b, t])
        lo = max(lo, hi - self.slots + 1)
        ring = [p % self.slots for p in range(lo, hi + 1)]
        if self.tk is None:
            return ring, []
        if self.mask is None:
            return ring, list(range(t + 1))
        return ring, [j for j in range(self.T) if (int(self.mask[b, t, j // 32]) >> (j % 32)) & 1]

    def want(self):
        f8 = np.float64
        out = np.zeros((self.B, self.T, self.heads, self.vh))
        tol = np.zeros((self.B, self.T, self.heads, 1))
        rep = self.heads // self.kvh
        for b in range(self.B):
            for t in range(self.T):
                ring, nodes = self.seen(b, t)
                if not ring and not nodes:
                    continue
                k, v = self.k[b, ring].astype(f8), self.v[b, ring].astype(f8)
                if self.int8:
                    k, v = k * self.ks[b, ring][..., None], v * self.vs[b, ring][..., None]
                if nodes:
                    dk, dv = self.tk[b, nodes].astype(f8), self.tv[b, nodes].astype(f8)
                    if self.int8:
                        dk, dv = dk * self.tks[b, nodes][..., None], dv * self.tvs[b, nodes][..., None]
                    k, v = np.concatenate([k, dk]), np.concatenate([v, dv])
                for h in range(self.heads):
                    qv = self.q[b, t, h * self.qk: (h + 1) * self.qk].astype(f8)
                    kh, vv = k[:, h // rep], v[:, h // rep]
                    s = kh @ qv / np.sqrt(self.qk)
                    w = np.exp(s - s.max())
                    out[b, t, h] = (w / w.sum()) @ vv
                    # A score: 2^-21 for the split query (and, f32, key) parts, 2^-23 per
                    # accumulation step (3 products per 8 dims at most) and per scaling, of
                    # sum |q k|; a weight follows it and adds 2^-21 (exponential, split);
                    # numerator and sum each take that error of the weights, and the
                    # running sums 2^-23 per 8 positions and merge.
                    size = (np.abs(kh) @ np.abs(qv)).max() / np.sqrt(self.qk)
                    ds = size * (2.0 ** -21 + 2.0 ** -23 * (3 * self.qk / 8 + 4))
                    tol[b, t, h] = np.abs(vv).max() * (2 * (ds + 2.0 ** -21) + 2.0 ** -23 * (len(s) / 4 + 16))
        return out, tol

    def run(self, torch, stream=None, out=None):
        d = {n: dev(torch, getattr(self, n)) for n in ("q", "k", "v", "ks", "vs", "lo", "hi", "tk", "tv", "tks", "tvs",
                                                       "mask")}
        self.keep = d
        if out is None:
            out = torch.full((self.B, self.T, self.heads, self.vh), 11.0, device="cuda")
        self.call(d, out, stream)
        return out

    def call(self, d, out, stream=None):
        nb.attend_tree(ptr(d["q"]), self.ldq, ptr(d["k"]), ptr(d["v"]), ptr(d["ks"]), ptr(d["vs"]), self.int8,
                       self.slots, ptr(d["lo"]), ptr(d["hi"]), ptr(d["tk"]), ptr(d["tv"]), ptr(d["tks"]),
                       ptr(d["tvs"]), ptr(d["mask"]), self.B, self.T, self.heads, self.kvh, self.qk, self.vh,
                       ptr(out), stream)

    def check(self, torch):
        got = self.run(torch).cpu().numpy()
        want, tol = self.want()
        assert np.isfinite(got).all()
        bad = np.abs(got - want) > tol
        assert not bad.any(), (np.argwhere(bad)[:4], float((np.abs(got - want) / np.maximum(tol, 1e-30)).max()))
        return got


SHAPES = [
    # B, T, heads, kv_heads, qk, vh, slots, ctx
    (1, 1, 1, 1, 16, 32, 1, 1),
    (3, 1, 12, 2, 48, 64, 100, 77),
    (2, 7, 12, 2, 48, 64, 130, 130),
    (2, 16, 12, 2, 48, 64, 300, 200),
    (1, 33, 6, 2, 64, 64, 90, 61),
    (2, 5, 4, 2, 16, 32, 8, 8),
    (1, 40, 8, 1, 48, 64, 40, 3),
    (2, 9, 16, 2, 128, 128, 70, 66),
    (1, 3, 3, 3, 20, 36, 50, 45),       # widths that are no multiple of 16
    (1, 12, 5, 1, 100, 12, 33, 30),
    (2, 4, 9, 1, 64, 64, 1500, 1403),   # split over the positions
    (1, 70, 2, 2, 48, 32, 700, 650),    # more than two mask words
    (1, 1, 40, 1, 128, 64, 2000, 1999),
]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_tree_attention_matches_64_bits(cuda, int8, shape):
    B, T, heads, kvh, qk, vh, slots, ctx = shape
    Tree(B, T, heads, kvh, qk, vh, slots, ctx, int8, seed=sum(shape), extra=3 if T % 2 else 0).check(cuda)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("qgain,vgain", [(1e-6, 1e-8), (6.0, 3e4), (1e4, 1.0)])
def test_tree_attention_over_the_range_of_values(cuda, int8, qgain, vgain):
    """Small and large queries and values; the last saturates on one position."""
    Tree(2, 6, 6, 2, 48, 64, 90, 80, int8, seed=5, qgain=qgain, vgain=vgain).check(cuda)


@pytest.mark.parametrize("int8", [False, True])
def test_tree_attention_without_a_draft_and_chains(cuda, int8):
    torch = cuda
    Tree(2, 3, 4, 2, 48, 64, 60, 50, int8, seed=1, drafted=False).check(torch)
    for T in (1, 5, 32, 45):
        Tree(2, T, 4, 2, 48, 64, 60, 50, int8, seed=T, mask="chain").check(torch)
    Tree(2, 5, 4, 2, 48, 64, 60, 0, int8, seed=3).check(torch)  # an empty ring: the draft alone


@pytest.mark.parametrize("int8", [False, True])
def test_tree_attention_ranges_of_their_own(cuda, int8):
    """Windows by depth, empty nodes, ranges longer than the ring and ranges far
    apart; a node that sees nothing gets zeros."""
    torch = cuda
    c = Tree(3, 8, 12, 2, 48, 64, 40, 30, int8, seed=9)
    for b in range(3):
        for t in range(8):
            c.lo[b, t] += 2 * t
    c.lo[0, 3], c.hi[0, 3] = 5, 4          # nothing of the ring
    c.mask[0, 3] = 0                       # and nothing of the draft
    c.lo[1, :], c.hi[1, :] = 0, 1000       # a thousand positions of a ring of 40
    c.lo[2, 0], c.hi[2, 0] = 3, 9
    c.lo[2, 1], c.hi[2, 1] = 100000, 100020
    c.lo[2, 2], c.hi[2, 2] = 2147483647 - 20, 2147483647
    c.lo[2, 3], c.hi[2, 3] = -50, 12       # positions below 0 do not exist
    c.lo[2, 4], c.hi[2, 4] = -50, -20
    got = c.check(torch)
    assert np.all(got[0, 3] == 0.0)
    c.hi[:] = -1
    c.mask[:] = 0
    assert np.all(c.check(torch) == 0.0)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), -3.4028234663852886e38])
def test_what_a_node_does_not_see_never_reaches_it(cuda, int8, bad):
    """Padding nodes and ring places out of range hold garbage: outputs of the
    others are the same as with zeros there, to the bit or within the bound."""
    torch = cuda
    c = Tree(2, 12, 12, 2, 48, 64, 64, 40, int8, seed=21)
    want, tol = c.want()
    pad = [9, 10, 11]                       # padding nodes: they see themselves only, no one sees them
    for t in range(12):
        for j in pad:
            c.mask[:, t] &= ~np.uint32(1 << j)
    for t in pad:
        c.mask[:, t] = np.uint32(1 << t)
    want, tol = c.want()
    for b in range(2):
        free = [s for s in range(64) if all(s not in c.seen(b, t)[0] for t in range(12))]
        for s in free:
            if int8:
                c.ks[b, s] = c.vs[b, s] = bad
            else:
                c.k[b, s] = c.v[b, s] = bad
        for j in pad:
            if int8:
                c.tks[b, j] = c.tvs[b, j] = bad
            else:
                c.tk[b, j] = c.tv[b, j] = bad
        c.q[b, 10] = bad
    got = c.run(torch).cpu().numpy()
    assert np.all(np.abs(got[:, :9] - want[:, :9]) <= tol[:, :9])
    # a value that is seen does reach it, and only its dimension
    if not int8 and bad != bad:
        d = Tree(1, 2, 4, 2, 48, 64, 20, 10, False, seed=2)
        want, tol = d.want()
        ring, _ = d.seen(0, 0)
        d.v[0, ring[3], 0, 5] = bad
        got = d.run(torch).cpu().numpy()
        hit = np.zeros(got.shape, bool)
        hit[0, :, :2, 5] = True
        assert np.all(np.isnan(got[hit])) and np.all((np.abs(got - want) <= tol)[~hit])
        d.v[0, ring[3], 0, 5] = np.inf
        assert np.all(d.run(torch).cpu().numpy()[hit] == np.inf)


@pytest.mark.parametrize("int8", [False, True])
def test_value_scales_that_differ_by_many_powers(cuda, int8):
    """Later blocks hold far larger and far smaller values than the first."""
    torch = cuda
    c = Tree(1, 3, 4, 2, 48, 64, 320, 320, int8, seed=4)
    for i, s in enumerate([1e-30, 1e-3, 1e12, 1e-12, 1.0, 1e20, 1e-20, 1e3, 1e-38, 1e18]):
        at = slice(32 * i, 32 * i + 32)
        if int8:
            c.vs[:, at] *= np.float32(s)
        else:
            c.v[:, at] *= np.float32(s)
    c.check(torch)
    c = Tree(1, 2, 4, 2, 48, 64, 64, 64, int8, seed=4)  # tiny values alone
    if int8:
        c.vs *= np.float32(1e-32)
        c.tvs *= np.float32(1e-32)
    else:
        c.v *= np.float32(1e-32)
        c.tv *= np.float32(1e-32)
    c.check(torch)


def test_tree_attention_unaligned_rings(cuda):
    """Ring and draft starts that are 4-byte aligned only."""
    torch = cuda
    for int8 in (False, True):
        c = Tree(2, 6, 4, 2, 48, 64, 50, 45, int8, seed=8)
        a = c.run(torch)
        d = dict(c.keep)
        hold = []
        for n in ("k", "v", "tk", "tv"):
            t = d[n]
            step = 4 // t.element_size()
            buf = torch.zeros(t.numel() + step, dtype=t.dtype, device="cuda")
            buf[step:] = t.reshape(-1)
            hold.append(buf)
            d[n] = buf[step:]
        out = torch.zeros_like(a)
        c.call(d, out)
        assert torch.equal(out, a)


def test_tree_attention_many_sessions(cuda):
    """More sessions than one grid axis holds, and the last ones are right."""
    torch = cuda
    B = 65537
    k = torch.randn(B, 2, 1, 16, device="cuda")
    v = torch.randn(B, 2, 1, 32, device="cuda")
    q = torch.randn(B, 1, 16, device="cuda")
    lo = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    hi = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    out = torch.zeros(B, 1, 1, 32, device="cuda")
    nb.attend_tree(ptr(q), 16, ptr(k), ptr(v), None, None, False, 2, ptr(lo), ptr(hi), None, None, None, None, None, B,
                   1, 1, 1, 16, 32, ptr(out))
    assert torch.all((out[:, 0, 0] - v[:, 0, 0]).abs() <= 4 * 2.0 ** -23 * v[:, 0, 0].abs())


def test_tree_attention_of_a_chain_is_the_decode_steps(cuda):
    """T drafted nodes of a chain against T single steps of nd_attend_step, each
    with the earlier nodes already in the ring."""
    torch = cuda
    for int8 in (False, True):
        c = Tree(4, 6, 12, 2, 48, 64, 96, 70, int8, seed=13, mask="chain")
        want, tol = c.want()
        got = c.run(torch).cpu().numpy()
        d = c.keep
        out = torch.zeros(4, 12 * 64, device="cuda")
        kc, vc = d["k"].clone(), d["v"].clone()
        ks, vs = (d["ks"].clone(), d["vs"].clone()) if int8 else (None, None)
        b = torch.arange(4, device="cuda")
        for t in range(6):
            at = (d["hi"][:, t].long() + 1 + t) % 96
            kc[b, at], vc[b, at] = d["tk"][:, t], d["tv"][:, t]
            if int8:
                ks[b, at], vs[b, at] = d["tks"][:, t], d["tvs"][:, t]
            hi = (d["hi"][:, t] + 1 + t).contiguous()
            q, lo = d["q"][:, t].contiguous(), d["lo"][:, t].contiguous()
            nb.attend_step(ptr(q), ptr(kc), ptr(vc), ptr(ks), ptr(vs), int8, 96, ptr(lo), ptr(hi), 4, 12, 2, 48, 64,
                           ptr(out))
            step = out.cpu().numpy().reshape(4, 12, 64)
            assert np.all(np.abs(step - got[:, t]) <= 2 * tol[:, t])


# ------------------------------------------------------------------ logits
def logits_ref(x, hist, off, gen, rep, pres, freq, bids, bvals, boff, keep, masked):
    """64-bit values, a bound of the f32 steps' error, and the picks."""
    y = x.astype(np.float64)
    size = np.abs(y)
    for r in range(len(y)):
        if hist is not None:
            h = hist[off[r]: off[r + 1]]
            h = np.unique(h[(h >= 0) & (h < y.shape[1])])
            if rep is not None:
                y[r, h] = np.where(y[r, h] > 0, y[r, h] / rep[r], y[r, h] * rep[r])
            size[r, h] = np.maximum(size[r, h], np.abs(y[r, h]))
            a = hist[(off if gen is None else gen)[r]: off[r + 1]]
            a = a[(a >= 0) & (a < y.shape[1])]
            ids, n = np.unique(a, return_counts=True)
            less = n * (0 if freq is None else float(freq[r])) + (0 if pres is None else float(pres[r]))
            y[r, ids] -= less
            size[r, ids] += np.abs(less)
        if bids is not None:
            for i in range(boff[r], boff[r + 1]):
                if 0 <= bids[i] < y.shape[1]:
                    y[r, bids[i]] += float(bvals[i])
                    size[r, bids[i]] += abs(float(bvals[i]))
        if keep is not None:
            y[r, ~keep[r]] = masked
            size[r, ~keep[r]] = 0.0
    return y, size


# One rounding (2^-24 of the sizes added) for the penalty, the count's product,
# its sum, their difference and each bias: below 8 in all here.
LOGIT_TOL = 8 * 2.0 ** -24


@pytest.mark.parametrize("rows,vocab,ld,ldo,off", [
    (1, 1, 1, 1, 0), (3, 5, 5, 9, 0), (4, 500, 500, 500, 0), (2, 1023, 1023, 1024, 1), (5, 4099, 4099, 4099, 0),
    (2, 8192, 8192, 8192, 0), (3, 33001, 33003, 33003, 2), (2, 70000, 70001, 70000, 0),
])
@pytest.mark.parametrize("parts", ["all", "mask", "history", "bias", "none"])
def test_logits_match_64_bits(cuda, rows, vocab, ld, ldo, off, parts):
    torch = cuda
    r = np.random.default_rng(vocab + rows)
    x = (r.normal(size=(rows, ld)) * 4).astype(np.float32)
    x[0, :vocab: 3] = 0.0
    hist = hoff = gen = rep = pres = freq = bids = bvals = boff = keep = None
    if parts in ("all", "history"):
        lens = r.integers(0, 900, rows)
        lens[-1] = 0
        hoff = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        hist = (r.random(hoff[-1]) ** 3 * vocab * 1.05 - 2).astype(np.int32)  # some ids below 0 or past the end
        gen = (hoff[:-1] + lens // 3).astype(np.int32) if parts == "all" else None
        rep, pres, freq = ((a + 0.9 * r.random(rows)).astype(np.float32) for a in (0.8, -0.3, -0.2))
    if parts in ("all", "bias"):
        n = r.integers(0, 80, rows)
        boff = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        bids = r.integers(-2, min(vocab + 3, 60), boff[-1]).astype(np.int32)  # ids repeat within a row
        bvals = r.normal(size=boff[-1]).astype(np.float32)
    if parts in ("all", "mask"):
        keep = r.random((rows, vocab)) < 0.3
        if rows > 2:
            keep[1] = False
    d = [dev(torch, a) for a in (hist, hoff, gen, rep, pres, freq, bids, bvals, boff)]
    mask = None if keep is None else dev(torch, nb.pack_mask(keep).view(np.int32))
    buf = torch.zeros(rows * ld + off, device="cuda")
    buf[off:] = dev(torch, x).reshape(-1)
    y = torch.full((rows, ldo), 8.0, device="cuda")
    picks = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    nb.logits_adjust(buf.data_ptr() + 4 * off, ld, rows, vocab, y.data_ptr(), ldo, *[ptr(t) for t in d], ptr(mask),
                     (vocab + 31) // 32, -1e9, picks.data_ptr())
    got = y.cpu().numpy()
    want, size = logits_ref(x[:, :vocab], hist, hoff, gen, rep, pres, freq, bids, bvals, boff, keep, -1e9)
    n_bias = 1 + (0 if bids is None else 80)
    assert np.all(got[:, vocab:] == 8.0)
    assert np.all(np.abs(got[:, :vocab] - want) <= (LOGIT_TOL + (n_bias - 1) * 2.0 ** -24) * size)
    assert np.array_equal(picks.cpu().numpy(), got[:, :vocab].argmax(1))  # the first maximum of what it wrote
    # in place, without picks: the same values
    nb.logits_adjust(buf.data_ptr() + 4 * off, ld, rows, vocab, buf.data_ptr() + 4 * off, ld, *[ptr(t) for t in d],
                     ptr(mask), (vocab + 31) // 32, -1e9)
    z = buf[off:].cpu().numpy().reshape(rows, ld)
    assert np.array_equal(z[:, :vocab], got[:, :vocab]) and np.array_equal(z[:, vocab:], x[:, vocab:])


def test_logits_special_values(cuda):
    """Infinities and NaN: a masked place is `masked` whatever it held; a NaN is
    never picked; rows with nothing to pick answer 0."""
    torch = cuda
    V = 300
    x = np.zeros((6, V), np.float32)
    x[0, 7], x[0, 9] = np.inf, np.nan
    x[1] = -np.inf
    x[2] = np.nan
    x[3, 5], x[3, 6] = np.nan, 2.0
    x[4] = -np.inf
    x[4, 200] = -5.0
    x[5, :] = 1.5
    keep = np.ones((6, V), bool)
    keep[0, [7, 9]] = False
    keep[5, :17] = False
    xd, m = dev(torch, x), dev(torch, nb.pack_mask(keep).view(np.int32))
    y, p = torch.empty(6, V, device="cuda"), torch.empty(6, dtype=torch.int32, device="cuda")
    nb.logits_adjust(ptr(xd), V, 6, V, ptr(y), V, mask_ptr=ptr(m), mask_ld=10, picks_ptr=ptr(p))
    got = y.cpu().numpy()
    want = np.where(keep, x, -np.inf)
    assert np.array_equal(got, want, equal_nan=True)
    assert p.cpu().tolist() == [0, 0, 0, 6, 200, 17]


def test_logits_biases_of_one_id_add_in_list_order(cuda):
    torch = cuda
    V, n = 64, 100
    r = np.random.default_rng(0)
    vals = (r.normal(size=n) * 10.0 ** r.integers(-4, 5, n)).astype(np.float32)
    x = dev(torch, np.zeros((1, V), np.float32))
    ids, v, off = dev(torch, np.full(n, 3, np.int32)), dev(torch, vals), dev(torch, np.array([0, n], np.int32))
    y = torch.empty(1, V, device="cuda")
    want = np.float32(0)
    for a in vals:
        want = np.float32(want + a)
    for _ in range(5):
        nb.logits_adjust(ptr(x), V, 1, V, ptr(y), V, bias_ids_ptr=ptr(ids), bias_vals_ptr=ptr(v), bias_off_ptr=ptr(off))
        assert float(y[0, 3]) == float(want)


def test_logits_many_rows(cuda):
    torch = cuda
    rows, V = 65600, 40
    x = torch.randn(rows, V, device="cuda")
    y, p = torch.empty_like(x), torch.empty(rows, dtype=torch.int32, device="cuda")
    nb.logits_adjust(ptr(x), V, rows, V, ptr(y), V, picks_ptr=ptr(p))
    assert torch.equal(x, y) and torch.equal(p.long(), x.argmax(1))


def test_logits_follow_the_grammar_mask_of_constrained_decoding(cuda, sp_fixture):
    """needle_tokenizer_tool_mask through pack_mask: the pick equals the host
    path's argmax of logits plus mask (v3_engine.rs:410-420)."""
    torch = cuda
    tok = nb.Tokenizer(sp_fixture["blob"])
    tools = '[{"name":"get_weather","description":"d","parameters":{"type":"object","properties":{"city":{"type":"string"}}}}]'
    V = 512
    r = np.random.default_rng(3)
    for written in (b"", b'{"name":"', b'{"name":"get_'):
        mask = tok.tool_mask(tools, written, V)
        x = (r.normal(size=(4, V)) * 5).astype(np.float32)
        xd, m = dev(torch, x), dev(torch, np.repeat(nb.pack_mask(mask)[None], 4, 0).view(np.int32))
        y, p = torch.empty(4, V, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
        nb.logits_adjust(ptr(xd), V, 4, V, ptr(y), V, mask_ptr=ptr(m), mask_ld=V // 32, masked=-1e9, picks_ptr=ptr(p))
        assert np.array_equal(p.cpu().numpy(), (x + mask).argmax(1))


# ------------------------------------------------------------------ streams, graphs, devices
def all_calls(torch, seed):
    """The five operators on small inputs: ([call(stream)], [output])."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = Tree(2, 8, 12, 2, 48, 64, 700, 640, True, seed=seed)
    out = c.run(torch)
    d = c.keep
    proj = torch.randn(16, 800, generator=g, device="cuda")
    y = torch.zeros(16, 672, device="cuda")
    pos = torch.arange(16, dtype=torch.int32, device="cuda") + 600
    sess = torch.arange(16, dtype=torch.int32, device="cuda") // 8
    kb, vb = torch.zeros(16, 96, device="cuda"), torch.zeros(16, 128, device="cuda")
    lg = torch.randn(16, 8192, generator=g, device="cuda")
    lo, pk = torch.zeros_like(lg), torch.zeros(16, dtype=torch.int32, device="cuda")
    off = torch.arange(17, dtype=torch.int32, device="cuda") * 4
    hist = torch.randint(0, 8192, (64,), generator=g, device="cuda", dtype=torch.int32)
    rep = torch.full((16,), 1.3, device="cuda")
    hold = (proj, pos, sess, hist, off, rep, lg, d)

    def rope(s):
        nb.rope(ptr(proj), 800, ptr(y), 672, ptr(pos), 16, 14, 48, stream=s)

    def append(s):
        nb.kv_append(ptr(proj) + 4 * 576, 800, ptr(proj) + 4 * 672, 800, ptr(sess), ptr(pos), 16, True, 2, 700, 2, 48,
                     64, ptr(d["k"]), ptr(d["v"]), ptr(d["ks"]), ptr(d["vs"]), stream=s)

    def read(s):
        nb.kv_read(ptr(d["k"]), ptr(d["v"]), ptr(d["ks"]), ptr(d["vs"]), True, 2, 700, 2, 48, 64, ptr(sess), ptr(pos),
                   16, ptr(kb), 96, ptr(vb), 128, stream=s)

    def tree(s):
        c.call(d, out, s)

    def logits(s):
        nb.logits_adjust(ptr(lg), 8192, 16, 8192, ptr(lo), 8192, hist_ptr=ptr(hist), hist_off_ptr=ptr(off),
                         repetition_ptr=ptr(rep), picks_ptr=ptr(pk), stream=s)

    return [rope, append, read, tree, logits], [y, kb, vb, out, lo, pk], hold


def test_streams_and_graphs_give_the_eager_results(cuda):
    """Two sets captured into two graphs, replayed together on two streams
    several times over, equal the eager calls to the bit."""
    torch = cuda
    sets = [all_calls(torch, s) for s in (1, 2)]
    want = []
    for calls, outs, _ in sets:
        for f in calls:
            f(None)
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for (calls, _, _), s in zip(sets, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for f in calls:
                f(s.cuda_stream)
        graphs.append(g)
    for _ in range(4):
        for calls, outs, _ in sets:
            for o in outs:
                o.fill_(3)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, outs, _), w in zip(sets, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, w))
    # eager on two streams at once
    for (calls, outs, _), s in zip(sets, streams):
        for o in outs:
            o.fill_(3)
    torch.cuda.synchronize()
    for _ in range(3):
        for (calls, _, _), s in zip(sets, streams):
            for f in calls:
                f(s.cuda_stream)
    torch.cuda.synchronize()
    for (_, outs, _), w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(outs, w))
    del graphs


def test_calls_repeat_to_the_bit(cuda):
    torch = cuda
    c = Tree(3, 10, 12, 2, 48, 64, 3000, 2900, True, seed=31)
    a = c.run(torch).clone()
    for _ in range(5):
        out = torch.zeros_like(a)
        c.call(c.keep, out)
        assert torch.equal(out, a)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("int8", [False, True])
def test_a_drafted_step_end_to_end(cuda, int8):
    """One layer of a server's step over a tree: rotate the projection's queries
    and keys at each node's depth, write the draft's keys and values, attend,
    then write the accepted path to the ring. The result equals decoding the
    accepted path token by token, and so does the ring, to the bit."""
    torch = cuda
    B, H, kvh, qk, vh, slots = 3, 12, 2, 48, 64, 64
    parents = [-1, 0, 0, 1, 3, 2, 4]
    path = [0, 1, 3, 4, 6]                 # the accepted nodes
    T, ctx = len(parents), [60, 13, 41]
    depth = [0] * T
    for t, p in enumerate(parents):
        depth[t] = depth[p] + 1 if p >= 0 else 0
    ld = (H + kvh) * qk + kvh * vh
    proj = torch.randn(B * T, ld, device="cuda")
    dt = torch.int8 if int8 else torch.float32

    def rings(n):
        k, v = (torch.zeros(B, n, kvh, w, dtype=dt, device="cuda") for w in (qk, vh))
        s = [torch.zeros(B, n, kvh, device="cuda") if int8 else None for _ in range(2)]
        return [k, v] + s

    ring, step_ring, draft = rings(slots), rings(slots), rings(T)
    past = torch.randn(sum(ctx), kvh * (qk + vh), device="cuda")
    ps = torch.tensor(np.repeat(np.arange(B), ctx), dtype=torch.int32, device="cuda")
    pp = torch.tensor(np.concatenate([np.arange(n) for n in ctx]), dtype=torch.int32, device="cuda")

    def append(src, lds, rows, sess, pos, to, n):
        nb.kv_append(src, lds, src + 4 * kvh * qk, lds, ptr(sess), ptr(pos), rows, int8, B, n, kvh, qk, vh, ptr(to[0]),
                     ptr(to[1]), ptr(to[2]), ptr(to[3]))

    for r in (ring, step_ring):
        append(past.data_ptr(), kvh * (qk + vh), len(past), ps, pp, r, slots)
    node = np.arange(B * T)
    at = torch.tensor([ctx[i // T] + depth[i % T] for i in node], dtype=torch.int32, device="cuda")
    sess = torch.tensor(node // T, dtype=torch.int32, device="cuda")
    slot = torch.tensor(node % T, dtype=torch.int32, device="cuda")
    rot = proj.clone()
    nb.rope(ptr(rot), ld, ptr(rot), ld, ptr(at), B * T, H + kvh, qk)  # queries and keys side by side, in place
    append(ptr(rot) + 4 * H * qk, ld, B * T, sess, slot, draft, T)
    lo = torch.zeros(B * T, dtype=torch.int32, device="cuda")
    hi = torch.tensor([ctx[i // T] - 1 for i in node], dtype=torch.int32, device="cuda")
    mask = dev(torch, np.repeat(nb.tree_mask(parents)[None], B, 0).view(np.int32))
    out = torch.zeros(B, T, H, vh, device="cuda")
    nb.attend_tree(ptr(rot), ld, ptr(ring[0]), ptr(ring[1]), ptr(ring[2]), ptr(ring[3]), int8, slots, ptr(lo), ptr(hi),
                   ptr(draft[0]), ptr(draft[1]), ptr(draft[2]), ptr(draft[3]), ptr(mask), B, T, H, kvh, qk, vh,
                   ptr(out))
    keep = torch.tensor([ctx[i // T] + depth[i % T] if i % T in path else -1 for i in node], dtype=torch.int32,
                        device="cuda")
    append(ptr(rot) + 4 * H * qk, ld, B * T, sess, keep, ring, slots)
    # token by token
    single = torch.zeros(B, 1, H, vh, device="cuda")
    for t in path:
        rows = proj.view(B, T, ld)[:, t].contiguous()
        pos = torch.tensor([n + depth[t] for n in ctx], dtype=torch.int32, device="cuda")
        nb.rope(ptr(rows), ld, ptr(rows), ld, ptr(pos), B, H + kvh, qk)
        append(ptr(rows) + 4 * H * qk, ld, B, None, pos, step_ring, slots)
        first = (pos - (slots - 1)).clamp(min=0)
        nb.attend_tree(ptr(rows), ld, *[ptr(r) for r in step_ring], int8, slots, ptr(first), ptr(pos), None, None, None, None, None, B, 1, H, kvh, qk,
                       vh, ptr(single))
        # the tree saw positions 0.. where the ring now starts one later per wrap: compare where nothing was dropped
        for b in range(B):
            if ctx[b] + depth[t] < slots:
                a, w = out[b, t], single[b, 0]
                # each within Tree.want's bound: sum |q k| / sqrt(qk) below 12 and values below
                # 5 here make it 5 * 2 * 12 * (2^-21 + 22 * 2^-23) = 3.8e-4 at most
                assert (a - w).abs().max() <= 2 * 3.8e-4
    for a, b in zip(ring, step_ring):
        assert (a is None and b is None) or torch.equal(a, b)


def test_the_workloads_agree_with_their_plain_forms(cuda):
    """perf/operators.py: small draws of every operator, kernels against the
    plain torch forms within f32 rounding of the whole output."""
    import random
    torch = cuda
    spec = importlib.util.spec_from_file_location("draft_workloads", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    rng, done = random.Random(7), {}
    while len(done) < 5 or min(done.values()) < 3:
        c = m.draw(rng)
        if done.get(c["op"], 0) >= 3 or m.work(c)["flops"] > 2e9:
            continue
        done[c["op"]] = done.get(c["op"], 0) + 1
        m.own = False
        want = m.run(m.prepare(c, 5))
        m.own = True
        got = m.run(m.prepare(c, 5))
        want, got = (x if isinstance(x, tuple) else (x,) for x in (want, got))
        for a, b in zip(got, want):
            if a.dtype == torch.int32:
                assert torch.equal(a, b), c
            else:
                a, b = a.reshape(-1).double(), b.reshape(-1).double()
                fin = torch.isfinite(b)
                assert torch.equal(a[~fin], b[~fin]) and float((a - b)[fin].norm()) <= 1e-5 * float(b[fin].norm()), c


@pytest.mark.parametrize("int8", [False, True])
def test_the_oracle_decode_agrees(cuda, int8):
    """One node over a wrapped ring against the CPU oracle's decode attention
    (attention.rs:300-377) on the same cache."""
    c = Tree(2, 1, 12, 2, 48, 64, 64, 60, int8, seed=77, drafted=False)
    got = c.run(cuda).cpu().numpy()
    _, tol = c.want()
    for b in range(2):
        kv = (dict(kq=c.k[b].ravel(), ks=c.ks[b].ravel(), vq=c.v[b].ravel(), vs=c.vs[b].ravel()) if int8 else
              dict(k=c.k[b].ravel(), v=c.v[b].ravel()))
        want = orc.attend_step(c.q[b, 0].ravel(), 64, int(c.lo[b, 0]), int(c.hi[b, 0]), 12, 2, 48, 64, **kv)
        # the oracle sums in f32 itself: within its own rounding, the bound again
        assert np.all(np.abs(got[b, 0] - np.asarray(want).reshape(12, 64)) <= 2 * tol[b, 0])
