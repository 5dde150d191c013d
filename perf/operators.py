"""Workloads of the operators for verifying drafted tokens over a quantised cache.

A server that drafts a tree of tokens per session and checks it in one forward
runs, per layer, rotary positions on the projected queries and keys
(nd_rope), the write of keys and values into a ring that may be int8
(nd_kv_append, read back with nd_kv_read) and attention of every drafted node
over the ring and its own ancestors (nd_attend_tree); after the last layer it
corrects the logits of every node (nd_logits_adjust). Each case here is one
call (for the append: the write and the read of what was written).

`run` computes a case with elementary torch operations where `own` is false
and through the package's entry points where it is true; `exact` computes the
same from the definitions in 64 bits.
"""
import math
import os

import torch

own = False

_pkg = None
MASKED = -math.inf  # what a forbidden token's logit becomes


def _nb():
    global _pkg
    if _pkg is None:
        import importlib.util
        import sys
        if "needle_b200" in sys.modules:
            _pkg = sys.modules["needle_b200"]
        else:
            d = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "needle-rs_b200")
            spec = importlib.util.spec_from_file_location("needle_b200", os.path.join(d, "__init__.py"),
                                                          submodule_search_locations=[d])
            mod = importlib.util.module_from_spec(spec)
            sys.modules["needle_b200"] = mod
            spec.loader.exec_module(mod)
            _pkg = mod
    return _pkg


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # The queries and keys of one decode step of 64 sessions at the shipped head
        # geometry (12 query and 2 key heads of 48, side by side in the projection's rows).
        dict(name="rope decode", op="rope", rows=64, heads=14, dim=48, rot=48, interleaved=False,
             scaling="none", far=2048, factor=1.0, ld=800),
        # A chunk of long prompts: interleaved pairs, half of the head rotated, positions far
        # past the trained context, frequencies stretched by parts.
        dict(name="rope long prompt", op="rope", rows=16384, heads=18, dim=64, rot=32, interleaved=True,
             scaling="by_parts", far=1 << 20, factor=32.0, ld=1216),
        # One new position of 64 sessions, full precision ring: the smallest write.
        dict(name="append f32 decode", op="append", int8=False, rows=64, sessions=64, slots=512, kv_heads=2,
             qk=48, vh=64, ld=800),
        # A prefill group of whole prompts into int8 rings (the engine's 16384-row forward).
        dict(name="append int8 prompt", op="append", int8=True, rows=16384, sessions=16, slots=1088, kv_heads=2,
             qk=48, vh=64, ld=800),
        # A short shared prefix read back from full precision rings.
        dict(name="read f32 prefix", op="read", int8=False, rows=256, sessions=8, slots=512, kv_heads=2, qk=48,
             vh=64),
        # The rings of 128 sessions read back whole (a cache moved or checked).
        dict(name="read int8 rings", op="read", int8=True, rows=133504, sessions=128, slots=1043, kv_heads=2, qk=48,
             vh=64),
        # One token of eight sessions: the step without a draft, where latency counts.
        dict(name="tree single token", op="tree", int8=True, B=8, T=1, heads=12, kv_heads=2, qk=48, vh=64, ctx=512,
             slots=1024, window=0),
        # 256 sessions checking 16-node trees at the benchmark's context, local window of 1024.
        dict(name="tree 16 nodes int8", op="tree", int8=True, B=256, T=16, heads=12, kv_heads=2, qk=48, vh=64,
             ctx=1043, slots=1088, window=1024),
        # Wide trees over full precision rings with odd lengths.
        dict(name="tree 48 nodes f32", op="tree", int8=False, B=16, T=48, heads=12, kv_heads=2, qk=48, vh=64,
             ctx=2051, slots=2304, window=0),
        # Few sessions with long contexts and 128-wide heads: work split over the positions.
        dict(name="tree long int8", op="tree", int8=True, B=4, T=32, heads=32, kv_heads=8, qk=128, vh=128, ctx=32771,
             slots=33000, window=0),
        # The nodes of one small tree at the shipped vocabulary, every correction on.
        dict(name="logits one tree", op="logits", rows=8, vocab=8192, hist=300, bias=16, mask=True),
        # 256 rows of a large odd vocabulary with histories of a thousand tokens.
        dict(name="logits large vocabulary", op="logits", rows=256, vocab=100003, hist=1043, bias=64, mask=True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "tree", "tree", "logits"])
    if op == "rope":
        dim = rng.choice([16, 32, 48, 64, 96, 128])
        rot = 2 * rng.randint(1, dim // 2)
        heads = rng.randint(1, 20)
        return dict(op=op, rows=_log(rng, 1, 8192), heads=heads, dim=dim, rot=rot,
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "by_parts"]),
                    far=_log(rng, 16, 1 << 20), factor=rng.choice([2.0, 8.0, 40.0]),
                    ld=heads * dim + rng.choice([0, 1, 32, 65]))
    if op in ("append", "read"):
        kv, qk, vh = rng.randint(1, 4), rng.choice([16, 32, 48, 64, 80, 128]), rng.choice([32, 64, 128])
        sessions = _log(rng, 1, 64)
        c = dict(op=op, int8=rng.random() < 0.6, rows=_log(rng, 1, 16384), sessions=sessions,
                 slots=_log(rng, 17, 1100), kv_heads=kv, qk=qk, vh=vh)
        if op == "append":
            c["slots"] = max(c["slots"], -(-c["rows"] // sessions))
            c["ld"] = kv * (qk + vh) + rng.choice([0, 1, 7, 64])
        return c
    if op == "tree":
        kv, rep = rng.choice([1, 2, 4]), rng.randint(1, 8)
        qk, vh = rng.choice([(16, 32), (32, 32), (48, 64), (64, 64), (80, 64), (128, 128)])
        T = _log(rng, 1, 64)
        ctx = _log(rng, 1, 6000)
        B = _log(rng, 1, max(1, min(128, int(4e7 / (ctx * T * rep * kv)))))
        return dict(op=op, int8=rng.random() < 0.6, B=B, T=T, heads=kv * rep, kv_heads=kv, qk=qk, vh=vh, ctx=ctx,
                    slots=ctx + rng.randint(0, 63), window=rng.choice([0, 0, 1 + ctx // 2]))
    vocab = _log(rng, 33, 100000)
    return dict(op=op, rows=_log(rng, 1, 128), vocab=vocab, hist=_log(rng, 1, 1500), bias=rng.choice([0, 1, 40]),
                mask=rng.random() < 0.7)


# ------------------------------------------------------------------ inputs
def _quantise(x):
    """The engine's int8 quantiser over the last axis: scale = absmax / 127 (1 for a zero
    vector), code = x * (1 / scale) in 32 bits, rounded half away from zero."""
    am = x.abs().amax(-1, keepdim=True)
    # tensor by tensor: a quotient by a Python number would be a product with its reciprocal
    scale = torch.where(am > 0, am / torch.full_like(am, 127.0), torch.ones_like(am))
    y = x * (torch.ones_like(scale) / scale)
    r = torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y))
    # y + 0.5 may round up to the next integer just below a half: the remainder says so.
    r = torch.where((y - torch.trunc(y)).abs() < 0.5, torch.trunc(y), r)
    return r.clamp(-128, 127).to(torch.int8), scale.squeeze(-1)


def _turns(c):
    """Rotation per position of every pair in turns, in 64 bits, and the factor of cos and sin."""
    rot, theta, factor, trained = c["rot"], 10000.0, c["factor"], 4096.0
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = torch.pow(torch.tensor(theta, dtype=torch.float64), -2.0 * i / rot) / (2.0 * math.pi)
    if c["scaling"] == "linear":
        return f / factor, 1.0
    if c["scaling"] == "by_parts":
        keep = ((trained * f - 1.0) / 31.0).clamp(0.0, 1.0)  # 1 turn .. 32 turns within the trained context
        return f * keep + f / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _tree_parents(T, g):
    """Parent of every node: -1 (the last accepted token) or an earlier node."""
    u = torch.rand(T, generator=g)
    return [-1 if t == 0 else max(-1, t - 1 - int(float(u[t]) * 4)) for t in range(T)]


def _mask_words(parents):
    T = len(parents)
    words = (T + 31) // 32
    rows, depth = [], []
    for t, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | (1 << t))
        depth.append(depth[p] + 1 if p >= 0 else 0)
    w = [[(r >> (32 * j)) & 0xFFFFFFFF for j in range(words)] for r in rows]
    w = [[x - (1 << 32) if x >= (1 << 31) else x for x in r] for r in w]
    return w, depth


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 17)
    gc = torch.Generator()
    gc.manual_seed(seed * 7919 + 18)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    st = dict(c=c)
    if c["op"] == "rope":
        st["x"] = rn(c["rows"], c["ld"])
        st["pos"] = torch.randint(0, c["far"], (c["rows"],), generator=g, device=dev, dtype=torch.int32)
        st["y"] = torch.empty(c["rows"], c["heads"] * c["dim"], device=dev)
        f, m = _turns(c)
        st["turns"], st["m"] = f.to(dev), m
        return st
    if c["op"] in ("append", "read"):
        S, n, kv, qk, vh, M = c["sessions"], c["slots"], c["kv_heads"], c["qk"], c["vh"], c["rows"]
        if c["int8"]:
            st["kc"], st["ks"] = _quantise(rn(S, n, kv, qk))
            st["vc"], st["vs"] = _quantise(rn(S, n, kv, vh))
        else:
            st["kc"], st["vc"], st["ks"], st["vs"] = rn(S, n, kv, qk), rn(S, n, kv, vh), None, None
        st["k"], st["v"] = torch.empty(M, kv * qk, device=dev), torch.empty(M, kv * vh, device=dev)
        i = torch.arange(M, device=dev)
        per = -(-M // S)
        start = torch.randint(0, 3 * n, (S,), generator=g, device=dev)
        if c["op"] == "append":  # the sessions' new positions one after another, wrapping in their rings
            st["x"] = rn(M, c["ld"]) * (0.2 + 2.0 * torch.rand(M, 1, generator=g, device=dev))
            st["sess"] = (i // per).to(torch.int32)
            st["pos"] = (start[i // per] + i % per).to(torch.int32)
        else:
            st["sess"] = (i % S).to(torch.int32)
            st["pos"] = (start[i % S] + i // S).to(torch.int32)
        return st
    if c["op"] == "tree":
        B, T, H, kv, qk, vh, n, ctx = (c[x] for x in ("B", "T", "heads", "kv_heads", "qk", "vh", "slots", "ctx"))
        st["q"] = rn(B, T, H, qk) * 1.5
        k, v, tk, tv = rn(B, n, kv, qk), rn(B, n, kv, vh), rn(B, T, kv, qk), rn(B, T, kv, vh)
        if c["int8"]:
            for name, x in (("k", k), ("v", v), ("tk", tk), ("tv", tv)):
                st[name], st[name + "s"] = _quantise(x)
        else:
            st.update(k=k, v=v, tk=tk, tv=tv, ks=None, vs=None, tks=None, tvs=None)
        # Ragged contexts of ctx * (0.75 .. 1) positions, at any phase of the ring.
        length = ctx - (torch.rand(B, generator=gc) * 0.25 * (ctx - 1)).to(torch.int64)
        first = torch.randint(0, 2 * n, (B,), generator=gc)
        trees = [_mask_words(_tree_parents(T, gc)) for _ in range(min(B, 8))]
        words = torch.tensor([trees[b % len(trees)][0] for b in range(B)], dtype=torch.int32)
        depth = torch.tensor([trees[b % len(trees)][1] for b in range(B)], dtype=torch.int64)
        last = first + length - 1
        lo = first[:, None].expand(B, T)
        if c["window"]:  # a node at depth d sees the window that ends at its own position
            lo = torch.maximum(lo, last[:, None] + 1 + depth - c["window"] + 1)
        st["lo"] = lo.to(torch.int32).contiguous().to(dev)
        st["hi"] = last[:, None].expand(B, T).to(torch.int32).contiguous().to(dev)
        st["mask"] = words.to(dev)
        st["out"] = torch.empty(B, T, H, vh, device=dev)
        st["span"] = int(length.max())
        return st
    R, V = c["rows"], c["vocab"]
    st["x"] = rn(R, V) * 3.0
    lens = torch.randint(0, c["hist"] + 1, (R,), generator=gc)
    lens[0] = c["hist"]
    off = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    total = int(off[-1])
    u = torch.rand(total, generator=g, device=dev)
    st["hist"] = (u.pow(4) * V).to(torch.int32).clamp(max=V - 1)  # few tokens repeat often
    st["off"] = off.to(torch.int32).to(dev)
    st["gen"] = (off[:-1] + lens // 2).to(torch.int32).to(dev)  # the prompt is the first half
    st["row"] = torch.repeat_interleave(torch.arange(R), lens).to(dev)
    st["rep"] = 1.0 + 0.5 * torch.rand(R, generator=g, device=dev)
    st["pres"] = 0.8 * torch.rand(R, generator=g, device=dev)
    st["freq"] = 0.5 * torch.rand(R, generator=g, device=dev)
    nb = c["bias"]
    st["bids"] = torch.randint(0, V, (R * nb,), generator=g, device=dev, dtype=torch.int32)
    st["bvals"] = rn(R * nb) * 4.0
    st["boff"] = (torch.arange(R + 1) * nb).to(torch.int32).to(dev)
    if c["mask"]:  # a grammar leaves about one token in eight
        keep = torch.rand(R, (V + 31) // 32 * 32, generator=g, device=dev) < 0.125
        bits = keep.view(R, -1, 32).to(torch.int64) << torch.arange(32, device=dev)
        w = bits.sum(-1)
        st["mask"] = torch.where(w >= (1 << 31), w - (1 << 32), w).to(torch.int32)
    else:
        st["mask"] = None
    st["y"], st["pick"] = torch.empty(R, V, device=dev), torch.empty(R, dtype=torch.int32, device=dev)
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["c"]["op"]
    if own:
        return {"rope": _rope_own, "append": _append_own, "read": _read_own, "tree": _tree_own,
                "logits": _logits_own}[op](state)
    return {"rope": _rope_plain, "append": _append_plain, "read": _read_plain, "tree": _tree_plain,
            "logits": _logits_plain}[op](state)


def _p(t):
    return None if t is None else t.data_ptr()


def _rope_own(s):
    nb, c = _nb(), s["c"]
    sc = None
    if c["scaling"] == "linear":
        sc = nb.RopeScaling("linear", c["factor"])
    elif c["scaling"] == "by_parts":
        sc = nb.RopeScaling("by_parts", c["factor"], trained=4096)
    nb.rope(_p(s["x"]), c["ld"], _p(s["y"]), c["heads"] * c["dim"], _p(s["pos"]), c["rows"], c["heads"], c["dim"],
            rot_dim=c["rot"], theta=10000.0, interleaved=c["interleaved"], scaling=sc)
    return s["y"]


def _rope_plain(s):
    c = s["c"]
    M, H, D, r = c["rows"], c["heads"], c["dim"], c["rot"]
    x = s["x"][:, : H * D].reshape(M, H, D)
    t = s["pos"].to(torch.float64)[:, None] * s["turns"]  # 64 bits: far positions
    a = ((t - torch.round(t)) * (2.0 * math.pi)).to(torch.float32)
    cos, sin = (torch.cos(a) * s["m"])[:, None], (torch.sin(a) * s["m"])[:, None]
    if c["interleaved"]:
        x1, x2 = x[..., 0:r:2], x[..., 1:r:2]
        rot = torch.stack([x1 * cos - x2 * sin, x1 * sin + x2 * cos], -1).reshape(M, H, r)
    else:
        x1, x2 = x[..., : r // 2], x[..., r // 2: r]
        rot = torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], -1)
    return torch.cat([rot, x[..., r:]], -1).reshape(M, H * D)


def _append_own(s):
    nb, c, x = _nb(), s["c"], s["x"]
    kv, qk, vh, M = c["kv_heads"], c["qk"], c["vh"], c["rows"]
    nb.kv_append(_p(x), c["ld"], _p(x) + 4 * kv * qk, c["ld"], _p(s["sess"]), _p(s["pos"]), M, c["int8"],
                 c["sessions"], c["slots"], kv, qk, vh, _p(s["kc"]), _p(s["vc"]), _p(s["ks"]), _p(s["vs"]))
    return _read_own(s)


def _append_plain(s):
    c, x = s["c"], s["x"]
    kv, qk, vh, M = c["kv_heads"], c["qk"], c["vh"], c["rows"]
    k, v = x[:, : kv * qk].reshape(M, kv, qk), x[:, kv * qk: kv * (qk + vh)].reshape(M, kv, vh)
    at = s["sess"].long() * c["slots"] + s["pos"].long() % c["slots"]
    if c["int8"]:
        (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
        s["ks"].view(-1, kv)[at] = ks
        s["vs"].view(-1, kv)[at] = vs
    else:
        kc, vc = k, v
    s["kc"].view(-1, kv, qk)[at] = kc
    s["vc"].view(-1, kv, vh)[at] = vc
    return _read_plain(s)


def _read_own(s):
    nb, c = _nb(), s["c"]
    kv, qk, vh = c["kv_heads"], c["qk"], c["vh"]
    nb.kv_read(_p(s["kc"]), _p(s["vc"]), _p(s["ks"]), _p(s["vs"]), c["int8"], c["sessions"], c["slots"], kv, qk, vh,
               _p(s["sess"]), _p(s["pos"]), c["rows"], _p(s["k"]), kv * qk, _p(s["v"]), kv * vh)
    return s["k"], s["v"]


def _read_plain(s):
    c = s["c"]
    kv, qk, vh, M = c["kv_heads"], c["qk"], c["vh"], c["rows"]
    at = s["sess"].long() * c["slots"] + s["pos"].long() % c["slots"]
    k, v = s["kc"].view(-1, kv, qk)[at].float(), s["vc"].view(-1, kv, vh)[at].float()
    if c["int8"]:
        k, v = k * s["ks"].view(-1, kv)[at][..., None], v * s["vs"].view(-1, kv)[at][..., None]
    return k.reshape(M, kv * qk), v.reshape(M, kv * vh)


def _tree_own(s):
    nb, c = _nb(), s["c"]
    nb.attend_tree(_p(s["q"]), c["heads"] * c["qk"], _p(s["k"]), _p(s["v"]), _p(s["ks"]), _p(s["vs"]), c["int8"],
                   c["slots"], _p(s["lo"]), _p(s["hi"]), _p(s["tk"]), _p(s["tv"]), _p(s["tks"]), _p(s["tvs"]),
                   _p(s["mask"]), c["B"], c["T"], c["heads"], c["kv_heads"], c["qk"], c["vh"], _p(s["out"]))
    return s["out"]


def _tree_plain(s):
    c = s["c"]
    B, T, H, kv, qk, vh, n = (c[x] for x in ("B", "T", "heads", "kv_heads", "qk", "vh", "slots"))
    rep = H // kv
    hi = s["hi"].long()
    p = hi[:, :1] - s["span"] + 1 + torch.arange(s["span"], device=hi.device)  # [B][span] positions, newest last
    at = (p % n + torch.arange(B, device=hi.device)[:, None] * n).reshape(-1)

    def rows(name, d):
        cache, drafted = s[name].view(B * n, kv, d)[at].view(B, -1, kv, d).float(), s["t" + name].float()
        if c["int8"]:
            cache = cache * s[name + "s"].view(B * n, kv)[at].view(B, -1, kv, 1)
            drafted = drafted * s["t" + name + "s"][..., None]
        return torch.cat([cache, drafted], 1).permute(0, 2, 1, 3)  # [B][kv][span + T][d]

    q = s["q"].view(B, T, kv, rep, qk).permute(0, 2, 3, 1, 4).reshape(B, kv, rep * T, qk)
    sc = torch.matmul(q, rows("k", qk).transpose(-1, -2)) * (1.0 / math.sqrt(qk))
    seen = (p[:, None, :] >= s["lo"].long()[..., None]) & (p[:, None, :] <= hi[..., None])
    j = torch.arange(T, device=hi.device)
    anc = (s["mask"][:, :, (j // 32)].long() >> (j % 32)) & 1
    ok = torch.cat([seen, anc.bool()], -1)[:, None, None].expand(B, kv, rep, T, -1).reshape(B, kv, rep * T, -1)
    sc = sc.masked_fill(~ok, -math.inf)
    m = sc.amax(-1, keepdim=True)
    w = torch.exp(sc - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w, rows("v", vh)) / torch.where(total > 0, total, torch.ones_like(total))
    return o.view(B, kv, rep, T, vh).permute(0, 3, 1, 2, 4).reshape(B, T, H, vh)


def _logits_own(s):
    nb, c = _nb(), s["c"]
    some = c["bias"] > 0
    nb.logits_adjust(_p(s["x"]), c["vocab"], c["rows"], c["vocab"], _p(s["y"]), c["vocab"], hist_ptr=_p(s["hist"]),
                     hist_off_ptr=_p(s["off"]), gen_from_ptr=_p(s["gen"]), repetition_ptr=_p(s["rep"]),
                     presence_ptr=_p(s["pres"]), frequency_ptr=_p(s["freq"]),
                     bias_ids_ptr=_p(s["bids"]) if some else None, bias_vals_ptr=_p(s["bvals"]) if some else None,
                     bias_off_ptr=_p(s["boff"]) if some else None, mask_ptr=_p(s["mask"]),
                     mask_ld=(c["vocab"] + 31) // 32, masked=MASKED, picks_ptr=_p(s["pick"]))
    return s["y"], s["pick"]


def _logits_plain(s):
    c, x = s["c"], s["x"]
    R, V = c["rows"], c["vocab"]
    at = s["row"] * V + s["hist"].long()
    one = torch.ones_like(at, dtype=torch.float32)
    made = (torch.arange(at.numel(), device=at.device) >= s["gen"].long()[s["row"]]).float()
    seen = torch.zeros(R * V, device=x.device).index_add_(0, at, one).view(R, V) > 0
    count = torch.zeros(R * V, device=x.device).index_add_(0, at, made).view(R, V)
    rep = s["rep"][:, None]
    y = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    y = y - (count * s["freq"][:, None] + (count > 0) * s["pres"][:, None])
    if c["bias"]:
        row = torch.arange(R, device=x.device).repeat_interleave(c["bias"])
        y = y + torch.zeros(R * V, device=x.device).index_add_(0, row * V + s["bids"].long(), s["bvals"]).view(R, V)
    if s["mask"] is not None:
        bit = torch.arange(32, device=x.device, dtype=torch.int32)
        keep = ((s["mask"][..., None] >> bit) & 1).view(R, -1)[:, :V].bool()
        y = torch.where(keep, y, torch.full_like(y, MASKED))
    first = torch.where(y == y.amax(-1, keepdim=True), torch.arange(V, device=x.device), V).amin(-1)
    return y, first.to(torch.int32)


# ------------------------------------------------------------------ what a pass needs
def work(case):
    c = case
    if c["op"] == "rope":
        n = c["rows"] * c["heads"] * c["dim"]
        return {"bytes": 8.0 * n + 4 * c["rows"], "flops": 3.0 * c["rows"] * c["heads"] * c["rot"]}
    if c["op"] in ("append", "read"):
        n = c["rows"] * c["kv_heads"] * (c["qk"] + c["vh"])
        ring = n + 8 * c["rows"] * c["kv_heads"] if c["int8"] else 4 * n
        # append: the rows in, the ring's bytes out, and for the read-back the ring's in and the rows out
        times = 2 if c["op"] == "append" else 1
        return {"bytes": float(times * (4 * n + ring) + 8 * c["rows"]), "flops": float(times * 2 * n)}
    if c["op"] == "tree":
        B, T, H, kv, qk, vh = (c[x] for x in ("B", "T", "heads", "kv_heads", "qk", "vh"))
        span = 0.875 * c["ctx"]  # the contexts are ragged: 0.75 to 1 of ctx
        span = min(span, c["window"]) if c["window"] else span
        per = kv * ((qk + vh) + 8 if c["int8"] else 4 * (qk + vh))
        return {"bytes": B * ((span + T) * per + T * H * 4.0 * (qk + vh) + 8 * T),
                "flops": 2.0 * B * T * H * (qk + vh) * (span + T / 2)}
    n = c["rows"] * c["vocab"]
    return {"bytes": 8.0 * n + (n / 8 if c["mask"] else 0) + c["rows"] * (4 * c["hist"] / 2 + 8 * c["bias"] + 28),
            "flops": 4.0 * n}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c, f8 = case, torch.float64
    if c["op"] == "rope":
        M, H, D, r = c["rows"], c["heads"], c["dim"], c["rot"]
        y = s["x"][:, : H * D].to(f8).reshape(M, H, D).clone()
        freq, m = torch.empty(r // 2, dtype=f8), 1.0
        for i in range(r // 2):
            w = 10000.0 ** (-2.0 * i / r)
            if c["scaling"] == "linear":
                w /= c["factor"]
            elif c["scaling"] == "by_parts":
                turns = 4096.0 * w / (2.0 * math.pi)
                keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
                w, m = w / c["factor"] * (1.0 - keep) + w * keep, 1.0 + 0.1 * math.log(c["factor"])
            freq[i] = w
        z = torch.polar(torch.full((M, r // 2), m, dtype=f8, device="cuda"), s["pos"].to(f8)[:, None] * freq.cuda())
        a = torch.arange(r // 2, device="cuda")
        a, b = (2 * a, 2 * a + 1) if c["interleaved"] else (a, a + r // 2)
        w = torch.complex(y[..., a], y[..., b]) * z[:, None]
        y[..., a], y[..., b] = w.real, w.imag
        return y.reshape(M, H * D)
    if c["op"] in ("append", "read"):
        kv, qk, vh, M = c["kv_heads"], c["qk"], c["vh"], c["rows"]
        got = []
        for at, d, cache, scale in ((0, qk, "kc", "ks"), (kv * qk, vh, "vc", "vs")):
            if c["op"] == "append":
                x = s["x"][:, at: at + kv * d].reshape(M, kv, d).to(f8)
                if c["int8"]:  # the scale and its reciprocal are held in 32 bits, and so is the product
                    am = x.abs().amax(-1, keepdim=True)
                    sc = torch.where(am > 0, am / 127.0, torch.ones_like(am)).float().to(f8)
                    y = (x * (1.0 / sc).float().to(f8)).float().to(f8)
                    x = (torch.floor(y.abs() + 0.5) * torch.sign(y)).clamp(-128, 127) * sc
            else:
                n = s["pos"].long() % c["slots"]
                x = s[cache][s["sess"].long(), n].to(f8)
                if c["int8"]:
                    x = x * s[scale][s["sess"].long(), n].to(f8)[..., None]
            got.append(x.reshape(M, kv * d))
        return tuple(got)
    if c["op"] == "tree":
        B, T, H, kv, qk, vh, n = (c[x] for x in ("B", "T", "heads", "kv_heads", "qk", "vh", "slots"))
        rep = H // kv
        lo, hi, words = s["lo"].cpu().tolist(), s["hi"].cpu().tolist(), s["mask"].cpu().tolist()
        out = torch.zeros(B, T, H, vh, dtype=f8, device="cuda")
        bit = torch.arange(T)
        for b in range(B):
            first, last = min(lo[b]), max(hi[b])
            at = torch.arange(first, last + 1, device="cuda")
            k, v = s["k"][b, at % n].to(f8), s["v"][b, at % n].to(f8)
            tk, tv = s["tk"][b].to(f8), s["tv"][b].to(f8)
            if c["int8"]:
                k, v = k * s["ks"][b, at % n].to(f8)[..., None], v * s["vs"][b, at % n].to(f8)[..., None]
                tk, tv = tk * s["tks"][b].to(f8)[..., None], tv * s["tvs"][b].to(f8)[..., None]
            k, v = torch.cat([k, tk]), torch.cat([v, tv])
            w = torch.tensor(words[b])[:, bit // 32] >> (bit % 32) & 1
            ok = torch.cat([(at >= s["lo"][b][:, None]) & (at <= s["hi"][b][:, None]), w.bool().cuda()], 1)
            for h in range(kv):
                q = s["q"][b, :, h * rep: (h + 1) * rep].to(f8)
                sc = (q @ k[:, h].T) / math.sqrt(qk)
                sc = torch.where(ok[:, None], sc, torch.full_like(sc, -math.inf))
                out[b, :, h * rep: (h + 1) * rep] = torch.nan_to_num(torch.softmax(sc, -1), nan=0.0) @ v[:, h]
        return out
    R, V = c["rows"], c["vocab"]
    y = s["x"].to(f8)
    off, gen = s["off"].cpu().tolist(), s["gen"].cpu().tolist()
    for r in range(R):
        ids, count = torch.unique(s["hist"][off[r]: off[r + 1]].long(), return_counts=True)
        rep = s["rep"][r].to(f8)
        y[r, ids] = torch.where(y[r, ids] > 0, y[r, ids] / rep, y[r, ids] * rep)
        ids, count = torch.unique(s["hist"][gen[r]: off[r + 1]].long(), return_counts=True)
        y[r, ids] -= s["freq"][r].to(f8) * count + s["pres"][r].to(f8)
        n = c["bias"]
        y[r].index_add_(0, s["bids"][r * n: (r + 1) * n].long(), s["bvals"][r * n: (r + 1) * n].to(f8))
        if s["mask"] is not None:
            v = torch.arange(V, device="cuda")
            y[r, (s["mask"][r].long()[v // 32] >> (v % 32)) & 1 == 0] = MASKED
    pick = torch.stack([torch.nonzero(y[r] == y[r].max())[0, 0] for r in range(R)]).to(torch.int32)
    return y, pick
