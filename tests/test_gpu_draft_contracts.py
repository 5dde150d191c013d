"""What the header promises of the operators for drafted tokens at the edges of
its wording: rows skipped inside a prompt longer than its ring, and the like.

Tolerances are those of the 64-bit references (Tree.want, ROPE_TOL, LOGIT_TOL)
where nothing else stands beside the comparison.
"""
import numpy as np
import pytest
from conftest import nb
from test_gpu_draft import dev, ptr, quant_ref

pytestmark = pytest.mark.gpu


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
