"""The operators of a step that verifies drafted tokens: vmlm_hip_rope_qk,
vmlm_hip_attention_tree_kv4, vmlm_hip_sample and vmlm_hip_tree_accept_kv4, each
against its plain form.

A case is a dict of plain values; `kind` names the operator. With `own` false,
`run` is the plain form in f32 torch operations (f64 where a border between two
tokens or the angle of a far position needs it); with `own` true it makes the
library's calls, on the library's own stream (a null stream), as a program without
streams of its own makes them.
"""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda"
BLOCK = 32  # channels that share a scale, and positions of one block of V codes
VOCAB = 122753


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token of a sequence that decodes alone
        dict(name="rope_one", kind="rope", rows=1, heads=36, kv=36, hd=64, rot=64, inter=False,
             scaling="none", first=1000, fused=True),
        # a chunk of a long conversation: neighbouring pairs of half a head, positions past
        # the trained length, q and k read out of fused q/k/v rows
        dict(name="rope_prompt", kind="rope", rows=2048, heads=32, kv=8, hd=128, rot=64,
             inter=True, scaling="bands", first=100000, fused=True),
        # one sequence checks 8 drafted tokens against a 1024-position cache
        dict(name="tree_one", kind="tree", batch=1, heads=36, kv=36, hd=64, cap=1024, first=1000,
             s=8, chain=False),
        # 16 slots of a serving loop with trees of up to 32 tokens, of other lengths, the last idle
        dict(name="tree_batch", kind="tree", batch=16, heads=36, kv=36, hd=64, cap=1024,
             first=960, s=32, chain=False),
        # one long context and a wide tree
        dict(name="tree_long", kind="tree", batch=1, heads=36, kv=36, hd=64, cap=65536,
             first=65400, s=63, chain=False),
        # grouped heads (4 queries a cache), 8 long conversations
        dict(name="tree_grouped", kind="tree", batch=8, heads=32, kv=8, hd=128, cap=16384,
             first=16000, s=16, chain=False),
        # a later chunk of three conversations: every token sees those before it
        dict(name="chunk", kind="tree", batch=3, heads=32, kv=8, hd=128, cap=4352, first=4000,
             s=333, chain=True),
        # one sequence's next token
        dict(name="sample_one", kind="sample", rows=1, vocab=VOCAB, spread=3.0, mix=False),
        # 16 sequences with settings of their own, some greedy, one slot idle
        dict(name="sample_batch", kind="sample", rows=16, vocab=VOCAB, spread=3.0, mix=True),
        # every node of 16 trees
        dict(name="sample_nodes", kind="sample", rows=512, vocab=VOCAB, spread=3.0, mix=True),
        # one sequence keeps what was accepted, two layers' caches
        dict(name="accept_one", kind="accept", batch=1, kv=36, hd=64, cap=1024, first=1000, s=8,
             layers=2),
        # 16 slots with wide trees, four layers' caches
        dict(name="accept_batch", kind="accept", batch=16, kv=36, hd=64, cap=1024, first=700, s=63,
             layers=4),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rope", "tree", "tree", "tree", "sample", "sample", "accept"))
    if kind == "sample":
        vocab = _log(rng, 300, VOCAB)
        return dict(kind=kind, rows=_log(rng, 1, min(512, 512 * VOCAB // vocab)), vocab=vocab,
                    spread=rng.choice((0.5, 2.0, 3.0, 5.0)), mix=rng.random() < 0.7)
    kv = rng.choice((1, 2, 4, 8, 12, 36))
    per = rng.choice((1, 1, 2, 4, 8))
    hd = rng.choice((64, 64, 128, 32, 256))
    if kind == "rope":
        hd = rng.choice((64, 64, 128, 32, 80, 96, 256))
        rows = _log(rng, 1, max(1, min(4096, 2048 * 40 * 128 // ((per + 1) * kv * hd))))
        return dict(kind=kind, rows=rows, heads=kv * per, kv=kv, hd=hd,
                    rot=rng.choice((hd, hd, hd // 2, hd // 4)), inter=rng.random() < 0.5,
                    scaling=rng.choice(("none", "linear", "bands", "ramp")),
                    first=rng.choice((0, 1000, 100000)), fused=rng.random() < 0.5)
    if kind == "accept":
        batch, s = _log(rng, 1, max(1, min(16, 16 * 36 * 64 // (kv * hd)))), rng.randint(1, 64)
        first = rng.randint(0, 900)
        return dict(kind=kind, batch=batch, kv=kv, hd=hd, first=first, s=s,
                    cap=BLOCK * (-(-(first + s) // BLOCK) + rng.randint(0, 8)),
                    layers=rng.randint(1, 4))
    chain = rng.random() < 0.3
    batch = _log(rng, 1, 32)
    s = _log(rng, 1, 400) if chain else rng.randint(1, 64)
    most = min(65400, 15 * 10 ** 7 // (batch * kv * hd),
               15 * 10 ** 9 // (batch * kv * per * hd * s))
    first = _log(rng, 1, max(2, most)) - 1
    return dict(kind="tree", batch=batch, heads=kv * per, kv=kv, hd=hd, first=first, s=s,
                cap=BLOCK * (-(-(first + s) // BLOCK) + rng.randint(0, 8)), chain=chain)


def _firsts(case):
    """Positions in each sequence's cache before the drafted tokens: from `first`
    down to half of it; of 8 slots or more, the last is idle."""
    b, top = case["batch"], case["first"]
    got = [top - (top // 2) * i // b for i in range(b)]
    if b >= 8:
        got[-1] = -1
    return got


def _counts(case):
    """Drafted tokens of each sequence: s, and fewer for the later ones."""
    return [max(1, case["s"] - (case["s"] // 3) * i // case["batch"]) for i in range(case["batch"])]


def _live(case):
    return [(f, n) for f, n in zip(_firsts(case), _counts(case)) if f >= 0]


def work(case):
    kind = case["kind"]
    if kind == "sample":
        return dict(bytes=4 * case["rows"] * case["vocab"] + 28 * case["rows"],
                    flops=4 * case["rows"] * case["vocab"])
    kv, hd = case["kv"], case["hd"]
    if kind == "rope":
        vals = case["rows"] * (case["heads"] + kv) * hd
        return dict(bytes=8 * vals + 4 * case["rows"], flops=3 * vals)
    if kind == "accept":
        # the window of drafted rows read, as far as it moved written, and read back in f32
        rows = 2 * kv * hd * case["layers"] * sum(n for _, n in _live(case))
        return dict(bytes=rows * 5 // 8 + 4 * rows, flops=2 * rows)
    seen = sum(f + n for f, n in _live(case))
    new = sum(n for _, n in _live(case))
    pairs = sum(n * f + n * (n + 1) // 2 for f, n in _live(case))
    return dict(bytes=seen * kv * hd * 2 * 5 // 8 + 8 * new * case["heads"] * hd,
                flops=4 * pairs * case["heads"] * hd)


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, dtype=torch.float32, generator=g)


def _rand(g, *shape):
    return torch.rand(*shape, device=DEV, dtype=torch.float32, generator=g)


def _ints(values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def _floats(values):
    return torch.tensor(values, device=DEV, dtype=torch.float32)


# A long context's scaling: base, factor, band edges and the length trained on
THETA, FACTOR, LOW, HIGH, TRAINED = 10000.0, 8.0, 1.0, 4.0, 8192.0


def _frequencies(case):
    """Radians a position for each pair, and the factor of the rotated values."""
    rot, kind = case["rot"], case["scaling"]
    f = THETA ** (-2.0 * np.arange(rot // 2) / rot)
    if kind == "linear":
        return f / FACTOR, 1.0
    if kind == "bands":  # long wavelengths are stretched, short ones kept
        turns = TRAINED * f / (2 * np.pi)
        keep = np.clip((turns - LOW) / (HIGH - LOW), 0.0, 1.0)
        return f * keep + f / FACTOR * (1 - keep), 1.0
    if kind == "ramp":  # the same along the pairs' indices
        at = [rot * np.log(TRAINED / (2 * np.pi * n)) / (2 * np.log(THETA)) for n in (HIGH, LOW)]
        lo, hi = max(np.floor(at[0]), 0.0), min(np.ceil(at[1]), rot - 1.0)
        away = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        return f * (1 - away) + f / FACTOR * away, 0.1 * math.log(FACTOR) + 1.0
    return f, 1.0


def _kv(g, batch, rows, kv, hd):
    """Keys (with channels that stand out, as trained ones have) and values of
    `rows` tokens, [batch][kv][rows][hd]."""
    k = _randn(g, batch, kv, rows, hd)
    k *= 1 + 3 * _rand(g, kv, 1, hd) ** 8
    k += _randn(g, kv, 1, hd) * 0.5
    return k, _randn(g, batch, kv, rows, hd)


def _cache(g, batch, kv, cap, hd):
    """A cache whose every position holds some token."""
    k, v = _kv(g, batch, cap, kv, hd)
    kc, km = _quantize(k)
    vc, vm = _quantize(v)
    return dict(k=_pack(kc), km=km, vm=vm,
                v=_pack(vc.unflatten(2, (-1, BLOCK)).transpose(-1, -2).contiguous()))


def _trees(rs, case):
    """parent [batch][s]: token 0 is the last one chosen (parent -1), the others hang
    below an earlier one, later ones rather below late ones, as a draft that goes deeper does."""
    got = np.full((case["batch"], case["s"]), -1, np.int32)
    for row in got:
        for t in range(1, case["s"]):
            row[t] = int(t * rs.random() ** 0.7)
    return got


def _accepting(rs, case):
    """Trees with drafted tokens and the tokens chosen at each, of which a path is
    accepted whose tokens after the first lie behind the rows that it will fill."""
    b, s = case["batch"], case["s"]
    parent = np.full((b, s), -1, np.int32)
    drafted = np.stack([rs.permutation(VOCAB // 2)[:s] for _ in range(b)]).astype(np.int32)
    chosen = (VOCAB // 2 + rs.integers(0, VOCAB // 2, (b, s))).astype(np.int32)
    for i, n in enumerate(_counts(case)):
        if n < 3:
            parent[i, 1:] = 0
            continue
        depth = int(rs.integers(1, max(2, int(math.sqrt(n)))))
        # the root's children, then levels below a level's last one and others
        wide = min(n - 1, depth + 1 + int(rs.integers(0, 3)))
        parent[i, 1:wide + 1] = 0
        path = [0, wide]
        for t in range(wide + 1, n):
            parent[i, t] = path[-1] if rs.random() < 0.5 or len(path) > depth else wide - 1
            if parent[i, t] == path[-1] and len(path) <= depth and rs.random() < 0.6:
                path.append(t)
        parent[i, n:] = 0
        for a, t in zip(path, path[1:]):
            chosen[i, a] = drafted[i, t]
    return parent, drafted, chosen


def _settings(rs, case):
    """Temperature, top-k, top-p and min-p of each row."""
    rows = case["rows"]
    if not case["mix"]:
        return [0.8] * rows, [50] * rows, [0.95] * rows, [0.0] * rows
    t = rs.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.5], rows).tolist()
    k = rs.choice([0, 0, 1, 40, 50, 1000], rows).tolist()
    p = rs.choice([1.0, 0.95, 0.9, 0.5, 1.0], rows).tolist()
    m = rs.choice([0.0, 0.0, 0.05, 0.2], rows).tolist()
    return t, k, p, m


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rs = np.random.default_rng(seed)
    kind = case["kind"]
    st = dict(case=case)
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = _randn(g, rows, vocab) * case["spread"]
        # the few tokens that a context makes likely, and for every fourth row a mask
        likely = torch.randint(0, vocab, (rows, 12), device=DEV, generator=g)
        logits.scatter_add_(1, likely, 3 * case["spread"] * _rand(g, rows, 12))
        banned = torch.randint(0, vocab, (rows, 64), device=DEV, generator=g)
        logits[::4].scatter_(1, banned[::4], -math.inf)
        u = _rand(g, rows)
        if case["mix"] and rows >= 8:
            u[-1] = -1.0  # an idle slot
        t, k, p, m = _settings(rs, case)
        st.update(logits=logits, u=u, t=_floats(t), k=_ints(k), p=_floats(p), m=_floats(m),
                  token=_ints([-1] * rows), prob=torch.zeros(rows, device=DEV))
    elif kind == "rope":
        rows, hd = case["rows"], case["hd"]
        wq, wk = case["heads"] * hd, case["kv"] * hd
        if case["fused"]:  # q and k lie in the rows of one projection, before v
            qkv = _randn(g, rows, wq + 2 * wk)
            st.update(q=qkv[:, :wq], k=qkv[:, wq:wq + wk])
        else:
            st.update(q=_randn(g, rows, wq), k=_randn(g, rows, wk))
        freq, factor = _frequencies(case)
        st.update(freq=torch.from_numpy(freq).to(DEV), factor=factor,
                  pos=torch.arange(rows, device=DEV, dtype=torch.int32) % 1024 + case["first"],
                  qo=torch.zeros(rows, wq, device=DEV), ko=torch.zeros(rows, wk, device=DEV))
    else:
        batch, s, kv, hd, cap = (case[x] for x in ("batch", "s", "kv", "hd", "cap"))
        st.update(pos0=_ints(_firsts(case)), count=_ints(_counts(case)))
        if kind == "tree":
            st.update(cache=_cache(g, batch, kv, cap, hd),
                      parent=None if case["chain"] else torch.from_numpy(_trees(rs, case)).to(DEV),
                      q=_randn(g, batch, s, case["heads"] * hd),
                      out=torch.zeros(batch, s, case["heads"] * hd, device=DEV))
        else:
            parent, drafted, chosen = (torch.from_numpy(x).to(DEV) for x in _accepting(rs, case))
            st.update(caches=[_cache(g, batch, kv, cap, hd) for _ in range(case["layers"])],
                      parent=parent, drafted=drafted, chosen=chosen,
                      path=torch.full_like(parent, -1), kept=_ints([0] * batch),
                      next=_ints([-1] * batch),
                      rows=[torch.zeros(batch, s, kv * hd, device=DEV)
                            for _ in range(2 * case["layers"])])
    torch.cuda.synchronize()
    return st


# ------------------------------------------------------------------ plain forms
def _nibbles(b):
    """The two codes of each byte, low one first, along the last axis: -8..7."""
    u = torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)
    return (u ^ 8).to(torch.int8) - 8


def _pack(q):
    """The inverse of _nibbles (q in -8..7)."""
    u = (q & 15).to(torch.uint8).unflatten(-1, (-1, 2))
    return u[..., 0] | (u[..., 1] << 4)


def _meta(m):
    """(scale, min) of 32 channels: bf16 bits in the low and the high half."""
    return (m << 16).view(torch.float32), (m & -65536).view(torch.float32)


def _quantize(x):
    """[..., hd] -> codes -8..7 and the packed (scale, min) of each 32 channels."""
    x = x.unflatten(-1, (-1, BLOCK))
    lo, hi = x.amin(-1), x.amax(-1)
    bits = lo.view(torch.int32)
    mn = torch.where(bits < 0, bits + 0xFFFF, bits) & -65536  # down to bf16
    low = mn.view(torch.float32)
    sc = (((hi - low) / 15).view(torch.int32) + 0xFFFF) & -65536  # up to bf16
    step = sc.view(torch.float32)[..., None]
    u = ((x - low[..., None]) / step).round().clamp(0, 15)
    return u.to(torch.int8).flatten(-2) - 8, mn | (sc >> 16 & 0xFFFF)


def _codes(cache):
    """Codes of the whole cache by position, [batch][kv][cap][hd] each."""
    v = _nibbles(cache["v"])  # [batch][kv][cap / 32][hd][32]
    return _nibbles(cache["k"]), v.transpose(-1, -2).flatten(2, 3)


def _values(codes, meta):
    scale, low = _meta(meta)
    u = codes.unflatten(-1, (-1, BLOCK)).float() + 8
    return (u * scale[..., None] + low[..., None]).flatten(-2)


def _plain_rope(st, x):
    case = st["case"]
    rot, x = case["rot"], x.unflatten(-1, (-1, case["hd"]))
    a = st["pos"].double()[:, None, None] * st["freq"]
    c, s = torch.cos(a).float() * st["factor"], torch.sin(a).float() * st["factor"]
    y = x.clone()
    if case["inter"]:
        lo, hi = x[..., :rot:2], x[..., 1:rot:2]
        y[..., :rot:2], y[..., 1:rot:2] = lo * c - hi * s, lo * s + hi * c
    else:
        h = rot // 2
        lo, hi = x[..., :h], x[..., h:rot]
        y[..., :h], y[..., h:rot] = lo * c - hi * s, lo * s + hi * c
    return y.flatten(-2)


def _ancestors(parent):
    """[batch][s][s]: whether token j is token t or above it."""
    b, s = parent.shape
    got = torch.eye(s, device=DEV, dtype=torch.bool).repeat(b, 1, 1)
    row = torch.arange(b, device=DEV)
    for t in range(1, s):
        got[:, t] |= got[row, parent[:, t].long().clamp(min=0)] & (parent[:, t] >= 0)[:, None]
    return got


def _plain_tree(st):
    case, cache = st["case"], st["cache"]
    batch, s, kv, hd, cap = (case[x] for x in ("batch", "s", "kv", "hd", "cap"))
    kc, vc = _codes(cache)
    k, v = _values(kc, cache["km"]), _values(vc, cache["vm"])
    q = st["q"].view(batch, s, kv, -1, hd).transpose(1, 2).reshape(batch, kv, -1, hd)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)
    at = torch.arange(cap, device=DEV)
    own_row = at - st["pos0"][:, None]  # the token that stands at a position
    if case["chain"]:
        seen = own_row[:, None] <= torch.arange(s, device=DEV)[:, None]
    else:
        above = _ancestors(st["parent"])
        seen = above.gather(2, own_row.clamp(0, s - 1)[:, None].expand(-1, s, -1))
        seen = (own_row < 0)[:, None] | (seen & (own_row < s)[:, None])
    per = case["heads"] // kv
    x = x.view(batch, kv, s, per, cap).masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p.view(batch, kv, -1, cap), v) / p.sum(-1).view(batch, kv, -1, 1)
    o = o.view(batch, kv, s, per, hd).transpose(1, 2).reshape(batch, s, -1)
    live = (torch.arange(s, device=DEV) < st["count"][:, None]) & (st["pos0"] >= 0)[:, None]
    st["out"].copy_(torch.where(live[..., None], o, st["out"]))
    return [st["out"]]


def _plain_sample(st):
    rows, vocab = st["logits"].shape
    x, order = torch.sort(st["logits"], dim=-1, descending=True, stable=True)
    greedy = st["t"] == 0
    t = torch.where(greedy, 1.0, st["t"]).double()
    w = torch.exp((x.double() - x[:, :1].double()) / t[:, None])
    rank = torch.arange(vocab, device=DEV)
    k = torch.where((st["k"] > 0) & (st["k"] < vocab), st["k"], vocab)
    k = torch.where(greedy, 1, k)
    w = torch.where(rank < k[:, None], w, 0.0)  # the k most likely
    c = torch.cumsum(w, -1)
    p = st["p"].double() * c[:, -1]
    inside = (c - w < p[:, None]) | (st["p"] >= 1)[:, None] | (rank == 0)
    inside &= w >= st["m"].double()[:, None]
    w = torch.where(inside, w, 0.0)
    c = torch.cumsum(w, -1)
    at = (c <= (st["u"].double() * c[:, -1])[:, None]).sum(-1, keepdim=True)
    at = at.clamp(max=vocab - 1)
    live = st["u"] >= 0
    token = order.gather(1, at)[:, 0].int()
    prob = (w.gather(1, at)[:, 0] / c[:, -1]).float()
    st["token"].copy_(torch.where(live, token, st["token"]))
    st["prob"].copy_(torch.where(live, prob, st["prob"]))
    return [st["token"], st["prob"]]


def _plain_accept(st):
    case = st["case"]
    batch, s = case["batch"], case["s"]
    at = torch.arange(s, device=DEV)
    live = st["pos0"] >= 0
    cur = torch.zeros(batch, device=DEV, dtype=torch.long)
    going = live.clone()
    path, kept = torch.full_like(st["parent"], -1), live.int()
    path[:, 0] = 0
    for i in range(1, s):
        want = st["chosen"].gather(1, cur[:, None])
        hit = (st["parent"] == cur[:, None]) & (st["drafted"] == want) & (at > cur[:, None])
        hit &= at < st["count"][:, None]
        going &= hit.any(-1)
        cur = torch.where(going, hit.int().argmax(-1), cur)
        path[:, i] = torch.where(going, cur.int(), -1)
        kept += going
    st["next"].copy_(torch.where(live, st["chosen"].gather(1, cur[:, None])[:, 0], st["next"]))
    st["kept"].copy_(torch.where(live, kept, st["kept"]))
    st["path"].copy_(torch.where(live[:, None], path, st["path"]))
    b, i = torch.nonzero((at < kept[:, None]) & live[:, None], as_tuple=True)
    dst = st["pos0"][b].long() + i
    src = st["pos0"][b].long() + path[b, i]
    rb, rt = torch.nonzero(live[:, None].expand(-1, s), as_tuple=True)
    rp = st["pos0"][rb].long() + rt
    for n, cache in enumerate(st["caches"]):
        kc, vc = _codes(cache)
        kc[b, :, dst], vc[b, :, dst] = kc[b, :, src], vc[b, :, src]
        for m in ("km", "vm"):
            cache[m][b, :, dst] = cache[m][b, :, src]
        cache["k"].copy_(_pack(kc))
        cache["v"].copy_(_pack(vc.unflatten(2, (-1, BLOCK)).transpose(-1, -2)))
        ko, vo = st["rows"][2 * n:2 * n + 2]
        ko[rb, rt] = _values(kc[rb, :, rp], cache["km"][rb, :, rp]).flatten(-2)
        vo[rb, rt] = _values(vc[rb, :, rp], cache["vm"][rb, :, rp]).flatten(-2)
    return [st["path"], st["kept"], st["next"], *st["rows"]]


# ------------------------------------------------------------------ the library's calls
def _p(t):
    return None if t is None else t.data_ptr()


@functools.cache
def _library():
    import sparrow_amd
    sparrow_amd.init(0)
    return sparrow_amd.lib(), sparrow_amd.check


def _descriptors(st):
    """The caches' descriptors, which a program makes once beside them."""
    if "desc" not in st:
        from sparrow_amd import _abi
        case, caches = st["case"], st["caches"] if "caches" in st else [st["cache"]]
        st["desc"] = (_abi.Kv4Cache * len(caches))(*(
            _abi.Kv4Cache(k=_p(c["k"]), v=_p(c["v"]), k_meta=_p(c["km"]), v_meta=_p(c["vm"]),
                          batch=case["batch"], n_kv_heads=case["kv"], cap=case["cap"],
                          head_dim=case["hd"]) for c in caches))
    return st["desc"]


def _own_rope(st):
    L, check = _library()
    case, q, k, qo, ko = st["case"], st["q"], st["k"], st["qo"], st["ko"]
    check(L.vmlm_hip_rope_qk(
        _p(qo), qo.stride(0), _p(ko), ko.stride(0), _p(q), q.stride(0), _p(k), k.stride(0),
        _p(st["pos"]), _p(st["freq"]), case["rows"], case["heads"], case["kv"], case["hd"],
        case["rot"], case["inter"], st["factor"], None))
    return [qo, ko]


def _own_tree(st):
    (L, check), desc, case = _library(), _descriptors(st), st["case"]
    w = case["heads"] * case["hd"]
    check(L.vmlm_hip_attention_tree_kv4(
        desc, _p(st["q"]), w, _p(st["pos0"]), _p(st["count"]), _p(st["parent"]), case["s"],
        _p(st["out"]), w, case["heads"], 1 / math.sqrt(case["hd"]), None, 0, None))
    return [st["out"]]


def _own_sample(st):
    L, check = _library()
    rows, vocab = st["logits"].shape
    check(L.vmlm_hip_sample(_p(st["logits"]), vocab, _p(st["u"]), _p(st["t"]), _p(st["k"]),
                            _p(st["p"]), _p(st["m"]), rows, vocab, _p(st["token"]),
                            _p(st["prob"]), None, 0, None))
    return [st["token"], st["prob"]]


def _own_accept(st):
    (L, check), desc, case = _library(), _descriptors(st), st["case"]
    s, w = case["s"], case["kv"] * case["hd"]
    check(L.vmlm_hip_tree_accept_kv4(
        desc, len(desc), _p(st["pos0"]), _p(st["count"]), _p(st["parent"]), _p(st["drafted"]),
        _p(st["chosen"]), s, _p(st["path"]), _p(st["kept"]), _p(st["next"]), None))
    for n in range(len(desc)):
        check(L.vmlm_hip_kv4_read(desc[n], _p(st["rows"][2 * n]), w, _p(st["rows"][2 * n + 1]), w,
                                  _p(st["pos0"]), None, s, None))
    return [st["path"], st["kept"], st["next"], *st["rows"]]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "tree": _own_tree, "sample": _own_sample,
                "accept": _own_accept}[kind](state)
    if kind == "rope":
        return [_plain_rope(state, state["q"]), _plain_rope(state, state["k"])]
    return {"tree": _plain_tree, "sample": _plain_sample, "accept": _plain_accept}[kind](state)


# ------------------------------------------------------------------ in 64 bits
def _split_bytes(b):
    """The codes 0..15 of bytes, low half first (f64)."""
    out = torch.empty(*b.shape[:-1], 2 * b.shape[-1], device=DEV, dtype=torch.float64)
    for half in range(2):
        out[..., half::2] = ((b.long() // 16 ** half % 16 + 8) % 16).double()
    return out


def _held(cache, b, n):
    """Keys and values of sequence b's first n positions, [kv][n][hd] in f64."""
    def wide(meta):  # (scale, min) of each channel; little-endian: the scale comes first
        ends = meta.view(torch.bfloat16).double().unflatten(-1, (-1, 2))
        return ends.repeat_interleave(BLOCK, dim=-2).unbind(-1)
    blocks = -(-n // BLOCK)
    ks, kl = wide(cache["km"][b, :, :n])
    vs, vl = wide(cache["vm"][b, :, :n])
    v = _split_bytes(cache["v"][b, :, :blocks]).permute(0, 1, 3, 2).flatten(1, 2)[:, :n]
    return kl + ks * _split_bytes(cache["k"][b, :, :n]), vl + vs * v


def _exact_rope(case, st):
    pos = st["pos"].cpu().numpy().astype(np.float64)
    turn = np.exp(1j * pos[:, None] * st["freq"].cpu().numpy()) * st["factor"]
    turn, rot, got = torch.from_numpy(turn).to(DEV)[:, None], case["rot"], []
    for x in (st["q"], st["k"]):
        y = x.double().reshape(case["rows"], -1, case["hd"])
        pair = y[..., :rot].unflatten(-1, (-1, 2) if case["inter"] else (2, -1))
        axis = -1 if case["inter"] else -2
        z = torch.complex(*(p.contiguous() for p in pair.unbind(axis))) * turn
        y = torch.cat((torch.stack((z.real, z.imag), axis).flatten(-2), y[..., rot:]), -1)
        got.append(y.reshape(case["rows"], -1))
    return got


def _exact_tree(case, st):
    heads, kv, hd = (case[x] for x in ("heads", "kv", "hd"))
    out = torch.zeros(case["batch"], case["s"], heads * hd, device=DEV, dtype=torch.float64)
    above = None if case["chain"] else st["parent"].tolist()
    for b, (first, n) in enumerate(zip(_firsts(case), _counts(case))):
        if first < 0:
            continue
        seen = np.zeros((n, first + n), bool)
        seen[:, :first] = True
        for t in range(n):  # up to the root, or along the chain
            at = t
            while at >= 0:
                seen[t, first + at] = True
                at = at - 1 if case["chain"] else above[b][at]
        seen = torch.from_numpy(seen).to(DEV)
        k, v = _held(st["cache"], b, first + n)
        q = st["q"][b, :n].double().view(n, heads, hd)
        for h in range(heads):
            j = h // (heads // kv)
            x = (q[:, h] @ k[j].T) * hd ** -0.5
            p = torch.softmax(torch.where(seen, x, -math.inf), -1)
            out[b, :n, h * hd:(h + 1) * hd] = p @ v[j]
    return [out]


def _exact_sample(case, st):
    token, prob = [], []
    columns = (st[x].cpu().numpy() for x in "utkpm")
    for row, (u, t, k, p, m) in enumerate(zip(*columns)):
        if u < 0:
            token.append(-1)
            prob.append(0.0)
            continue
        x = st["logits"][row].cpu().numpy().astype(np.float64)
        order = np.lexsort((np.arange(x.size), -x))
        if t == 0:
            token.append(order[0])
            prob.append(1.0)
            continue
        if 0 < k < x.size:
            order = order[:k]
        w = np.exp((x[order] - x[order[0]]) / np.float64(t))
        if p < 1:  # as many as it takes to reach p
            w = w[:1 + np.count_nonzero(np.cumsum(w)[:-1] < np.float64(p) * w.sum())]
        w = w[w >= np.float64(m)]
        c = np.cumsum(w)
        i = min(int(np.searchsorted(c, np.float64(u) * c[-1], side="right")), w.size - 1)
        token.append(order[i])
        prob.append(w[i] / c[-1])
    return [_ints([int(x) for x in token]), torch.tensor(prob, device=DEV, dtype=torch.float64)]


def _exact_accept(case, st):
    b, s, kv, hd = (case[x] for x in ("batch", "s", "kv", "hd"))
    parent, drafted, chosen = (st[x].tolist() for x in ("parent", "drafted", "chosen"))
    path, kept, nxt = [[-1] * s for _ in range(b)], [0] * b, [-1] * b
    rows = [torch.zeros(b, s, kv * hd, device=DEV, dtype=torch.float64) for _ in st["rows"]]
    for i, (first, n) in enumerate(zip(_firsts(case), _counts(case))):
        if first < 0:
            continue
        taken = [0]
        while True:
            below = [t for t in range(taken[-1] + 1, n) if parent[i][t] == taken[-1]
                     and drafted[i][t] == chosen[i][taken[-1]]]
            if not below:
                break
            taken.append(below[0])
        path[i][:len(taken)], kept[i], nxt[i] = taken, len(taken), chosen[i][taken[-1]]
        source = [first + t for t in taken + list(range(len(taken), s))]
        for c, cache in enumerate(st["caches"]):
            for j, x in enumerate(_held(cache, i, first + s)):
                rows[2 * c + j][i] = x[:, source].transpose(0, 1).flatten(1)
    return [_ints(path), _ints(kept), _ints(nxt), *rows]


def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "tree": _exact_tree, "sample": _exact_sample,
            "accept": _exact_accept}[case["kind"]](case, st)
