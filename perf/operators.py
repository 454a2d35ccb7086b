"""The operators of a decode layer with 4-bit weights and a 4-bit KV cache:
vmlm_hip_gemm_nt_int4, vmlm_hip_qk_norm_rope, vmlm_hip_kv4_append with
vmlm_hip_kv4_read, and vmlm_hip_attention_decode_kv4, each against its plain
form.

A case is a dict of plain values; `kind` names the operator. With `own` false,
`run` is the plain form in f32 torch operations; with `own` true it makes the
library's calls, on the library's own stream (a null stream), as a program
without streams of its own makes them.
"""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda"
THETA = 10000.0
EPS = 1e-5
BLOCK = 32  # channels that share a scale, and positions of one block of V codes


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one sequence's decode step: the o projection, launch latency and one
        # read of the weights
        dict(name="linear_one", kind="linear", m=1, n=2304, k=2304, group=128),
        # 16 sequences decoding together, a layer whose width is no multiple of
        # a tile, the finest scales
        dict(name="linear_batch", kind="linear", m=16, n=1537, k=992, group=32),
        # the LM head for one sequence
        dict(name="head_one", kind="linear", m=1, n=122753, k=2304, group=64),
        # the down projection of a prompt of 100 tokens
        dict(name="linear_prompt", kind="linear", m=100, n=2304, k=5760, group=128),
        # head norms and rotation of one decode token
        dict(name="norm_one", kind="norm", rows=1, heads=36, kv=36, hd=64, first=1000, fused=True),
        # the same for 16 prompts of 128 tokens, read out of fused q/k/v rows
        dict(name="norm_prompt", kind="norm", rows=2048, heads=36, kv=36, hd=64, first=0,
             fused=True),
        # the prompts' keys and values into the cache, and back as the values it holds
        dict(name="cache_prompt", kind="cache", batch=16, kv=36, hd=64, cap=1024, s=128, first=0),
        # a later chunk of three conversations of other lengths, from positions inside a block
        dict(name="cache_chunk", kind="cache", batch=3, kv=8, hd=128, cap=2048, s=333, first=1001),
        # one decode token against a 1024-position cache
        dict(name="attn_one", kind="attn", batch=1, heads=36, kv=36, hd=64, cap=1024, length=1024,
             append=True),
        # 16 slots of a serving loop, of other lengths, the last one idle
        dict(name="attn_batch", kind="attn", batch=16, heads=36, kv=36, hd=64, cap=1024,
             length=1000, append=True),
        # one sequence at a long context
        dict(name="attn_long", kind="attn", batch=1, heads=36, kv=36, hd=64, cap=65536,
             length=65500, append=False),
        # grouped heads (4 queries a cache), 8 long conversations
        dict(name="attn_grouped", kind="attn", batch=8, heads=32, kv=8, hd=128, cap=16384,
             length=16000, append=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "norm", "cache", "attn", "attn"))
    if kind == "linear":
        n = _log(rng, 64, 122753)
        m = _log(rng, 1, 100 if n < 6000 else 16)
        group = rng.choice((32, 64, 128, 128, 256, 0))
        k = BLOCK * _log(rng, 2, 180 if n < 6000 else 72)
        if m * n * k > 100 * 2304 * 5760:
            m = max(1, 100 * 2304 * 5760 // (n * k))
        return dict(kind=kind, m=m, n=n, k=k, group=group or -(-k // 128) * 128)
    kv = rng.choice((1, 2, 4, 8, 12, 36))
    per = rng.choice((1, 1, 2, 4, 8))
    hd = rng.choice((64, 64, 128, 32, 256))
    if kind == "norm":
        hd = rng.choice((64, 64, 128, 32, 80, 96, 256))
        rows = _log(rng, 1, max(1, min(4096, 2048 * 72 * 64 // ((per + 1) * kv * hd))))
        return dict(kind=kind, rows=rows, heads=kv * per, kv=kv, hd=hd,
                    first=rng.choice((0, 1000, 100000)), fused=rng.random() < 0.5)
    if kind == "cache":
        batch = _log(rng, 1, 16)
        s = _log(rng, 1, max(1, min(1024, 16 * 128 * 36 * 64 // (batch * kv * hd))))
        first = rng.choice((0, 0, rng.randint(1, 1000)))
        return dict(kind=kind, batch=batch, kv=kv, hd=hd, s=s, first=first,
                    cap=BLOCK * (-(-(s + first) // BLOCK) + rng.randint(0, 8)))
    batch = _log(rng, 1, 32)
    most = max(64, 8 * 8 * 12000 * 128 // (batch * kv * hd * max(1, per // 4)))
    length = _log(rng, 1, min(65536, most))
    return dict(kind=kind, batch=batch, heads=kv * per, kv=kv, hd=hd, length=length,
                cap=BLOCK * (-(-length // BLOCK) + rng.randint(0, 8)), append=rng.random() < 0.6)


def _lengths(case):
    """Positions per sequence after the call: from `length` down to half of it;
    of 8 slots or more, the last is idle (0)."""
    b, top = case["batch"], case["length"]
    got = [max(1, top - (top // 2) * i // b) for i in range(b)]
    if b >= 8:
        got[-1] = 0
    return got


def work(case):
    kind = case["kind"]
    if kind == "linear":
        m, n, k, g = (case[x] for x in ("m", "n", "k", "group"))
        return dict(bytes=n * k // 2 + 4 * n * -(-k // g) + 4 * m * k + 4 * m * n,
                    flops=2 * m * n * k)
    hd = case["hd"]
    if kind == "norm":
        vals = case["rows"] * (case["heads"] + case["kv"]) * hd
        return dict(bytes=8 * vals + 4 * case["rows"] + 8 * hd, flops=8 * vals)
    if kind == "cache":
        vals = 2 * sum(_counts(case)) * case["kv"] * hd
        # appended (f32 in, 5 bits out) and read back (5 bits in, f32 out)
        return dict(bytes=2 * (4 * vals + vals * 5 // 8), flops=8 * vals)
    lens = _lengths(case)
    live = sum(n > 0 for n in lens)
    moved = sum(lens) * case["kv"] * hd * 2 * 5 // 8 + 8 * live * case["heads"] * hd
    if case["append"]:
        moved += live * case["kv"] * hd * 2 * (8 + 5 / 8)  # new rows in, and back as they stand
    return dict(bytes=moved, flops=4 * sum(lens) * case["heads"] * hd)


def _counts(case):
    """Rows that each sequence appends: s, and fewer for the later ones."""
    return [max(1, case["s"] - 5 * i) for i in range(case["batch"])]


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, dtype=torch.float32, generator=g)


def _ints(values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def _kv(g, batch, rows, kv, hd):
    """Keys (with channels that stand out, as trained ones have) and values of
    `rows` tokens, [batch][rows][kv * hd]."""
    k = _randn(g, batch, rows, kv, hd) * (1 + 3 * torch.rand(kv, hd, device=DEV, generator=g) ** 8)
    k += _randn(g, kv, hd) * 0.5
    return k.view(batch, rows, kv * hd), _randn(g, batch, rows, kv * hd)


def _empty_cache(batch, kv, cap, hd):
    z = lambda *s, dt=torch.uint8: torch.zeros(*s, device=DEV, dtype=dt)  # noqa: E731
    return dict(k=z(batch, kv, cap, hd // 2), v=z(batch, kv, cap // BLOCK, hd, BLOCK // 2),
                km=z(batch, kv, cap, hd // BLOCK, dt=torch.int32),
                vm=z(batch, kv, cap, hd // BLOCK, dt=torch.int32))


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind = case["kind"]
    st = dict(case=case)
    if kind == "linear":
        m, n, k, group = (case[x] for x in ("m", "n", "k", "group"))
        st.update(a=_randn(g, m, k),
                  q=torch.randint(0, 256, (n, k // 2), device=DEV, dtype=torch.uint8, generator=g),
                  s=_randn(g, n, -(-k // group)).abs() * (0.02 / 7) + 1e-5,
                  c=torch.zeros(m, n, device=DEV))
    elif kind == "norm":
        rows, hd = case["rows"], case["hd"]
        wq, wk = case["heads"] * hd, case["kv"] * hd
        if case["fused"]:  # q and k lie in the rows of one projection, before v
            qkv = _randn(g, rows, wq + 2 * wk)
            st.update(q=qkv[:, :wq], k=qkv[:, wq:wq + wk])
        else:
            st.update(q=_randn(g, rows, wq), k=_randn(g, rows, wk))
        st.update(gq=1 + 0.1 * _randn(g, hd), gk=1 + 0.1 * _randn(g, hd),
                  pos=torch.arange(rows, device=DEV, dtype=torch.int32) % 1024 + case["first"],
                  qo=torch.zeros(rows, wq, device=DEV), ko=torch.zeros(rows, wk, device=DEV))
    else:
        batch, kv, hd, cap = (case[x] for x in ("batch", "kv", "hd", "cap"))
        cache = _empty_cache(batch, kv, cap, hd)
        # what the slots hold: earlier tokens, and behind them those of earlier conversations
        k, v = _kv(g, batch, cap, kv, hd)
        zero = torch.zeros(batch, device=DEV, dtype=torch.int32)
        _store(cache, k, v, zero, torch.full_like(zero, cap))
        del k, v
        if kind == "cache":
            k, v = _kv(g, batch, case["s"], kv, hd)
            st.update(first=_ints([case["first"]] * batch), count=_ints(_counts(case)))
        else:
            k, v = _kv(g, batch, 1, kv, hd)
            st.update(pos=_ints([n - 1 for n in _lengths(case)]),
                      q=_randn(g, batch, case["heads"] * hd),
                      out=torch.zeros(batch, case["heads"] * hd, device=DEV))
        st.update(cache=cache, k=k, v=v, ko=torch.zeros_like(k), vo=torch.zeros_like(v))
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


def _over(x, y):
    """x / y, rounded once to f32 (next to a border it decides a code)."""
    return (x.double() / y).float()


def _quantize(x):
    """[..., hd] -> codes -8..7 and the packed (scale, min) of each 32 channels."""
    x = x.unflatten(-1, (-1, BLOCK))
    lo, hi = x.amin(-1), x.amax(-1)
    bits = lo.view(torch.int32)
    mn = torch.where(bits < 0, bits + 0xFFFF, bits) & -65536  # down to bf16
    low = mn.view(torch.float32)
    sc = (_over(hi - low, 15.0).view(torch.int32) + 0xFFFF) & -65536  # up to bf16
    step = sc.view(torch.float32)[..., None]
    u = torch.where(step > 0, _over(x - low[..., None], step).round().clamp(0, 15), 0.0)
    return u.to(torch.int8).flatten(-2) - 8, mn | (sc >> 16 & 0xFFFF)


def _codes(cache):
    """Codes of the whole cache by position, [batch][kv][cap][hd] each."""
    v = _nibbles(cache["v"])  # [batch][kv][cap / 32][hd][32]
    return _nibbles(cache["k"]), v.transpose(-1, -2).flatten(2, 3)


def _rows(batch, s, pos0, count):
    """(sequence, row, position) of the rows that are live."""
    t = torch.arange(s, device=DEV)
    b, t = torch.nonzero((t < count[:, None]) & (pos0[:, None] >= 0), as_tuple=True)
    return b, t, pos0[b].long() + t


def _store(cache, k, v, pos0, count):
    batch, kv, cap = cache["k"].shape[:3]
    b, t, p = _rows(batch, k.shape[1], pos0, count)
    kc, vc = _codes(cache)
    for_each = lambda x: x[b, t].unflatten(-1, (kv, -1))  # noqa: E731
    kc[b, :, p], cache["km"][b, :, p] = _quantize(for_each(k))
    vc[b, :, p], cache["vm"][b, :, p] = _quantize(for_each(v))
    cache["k"].copy_(_pack(kc))
    cache["v"].copy_(_pack(vc.unflatten(2, (-1, BLOCK)).transpose(-1, -2)))


def _values(codes, meta, dtype=torch.float32):
    scale, low = _meta(meta)
    u = codes.unflatten(-1, (-1, BLOCK)).to(dtype) + 8
    return (u * scale[..., None].to(dtype) + low[..., None].to(dtype)).flatten(-2)


def _load(cache, ko, vo, pos0, count):
    b, t, p = _rows(ko.shape[0], ko.shape[1], pos0, count)
    kc, vc = _codes(cache)
    ko[b, t] = _values(kc[b, :, p], cache["km"][b, :, p]).flatten(-2)
    vo[b, t] = _values(vc[b, :, p], cache["vm"][b, :, p]).flatten(-2)


def _plain_linear(st):
    w = _nibbles(st["q"]).to(torch.float32)
    n, k = w.shape
    s = st["s"].repeat_interleave(st["case"]["group"], dim=1)[:, :k]
    return st["a"] @ (w * s).T


def _plain_norm(x, g, pos, hd):
    x = x.unflatten(-1, (-1, hd))
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * g
    i = torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    a = pos.to(torch.float64)[:, None, None] * THETA ** (-2 * i / hd)
    c, s = torch.cos(a).float(), torch.sin(a).float()
    lo, hi = y[..., :hd // 2], y[..., hd // 2:]
    return torch.cat((lo * c - hi * s, lo * s + hi * c), dim=-1).flatten(-2)


def _plain_attn(st):
    case, cache = st["case"], st["cache"]
    batch, kv, hd = case["batch"], case["kv"], case["hd"]
    if case["append"]:
        one = torch.ones_like(st["pos"])
        _store(cache, st["k"], st["v"], st["pos"], one)
        _load(cache, st["ko"], st["vo"], st["pos"], one)
    kc, vc = _codes(cache)
    k, v = _values(kc, cache["km"]), _values(vc, cache["vm"])
    q = st["q"].view(batch, kv, -1, hd)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)
    live = torch.arange(case["cap"], device=DEV) <= st["pos"][:, None]
    s = s.masked_fill(~live[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    st["out"].copy_(torch.where(st["pos"][:, None] >= 0, o.reshape(batch, -1), st["out"]))
    return [st["out"], st["ko"], st["vo"]] if case["append"] else [st["out"]]


# ------------------------------------------------------------------ the library's calls
def _p(t):
    return t.data_ptr()


@functools.cache
def _library():
    import sparrow_amd
    sparrow_amd.init(0)
    return sparrow_amd.lib(), sparrow_amd.check


def _descriptor(st):
    """The cache's descriptor, which a program makes once beside the cache."""
    if "desc" not in st:
        from sparrow_amd import _abi
        c, case = st["cache"], st["case"]
        st["desc"] = _abi.Kv4Cache(k=_p(c["k"]), v=_p(c["v"]), k_meta=_p(c["km"]),
                                   v_meta=_p(c["vm"]), batch=case["batch"],
                                   n_kv_heads=case["kv"], cap=case["cap"], head_dim=case["hd"])
    return st["desc"]


def _own_linear(st):
    L, check = _library()
    case = st["case"]
    check(L.vmlm_hip_gemm_nt_int4(_p(st["a"]), _p(st["q"]), _p(st["s"]), _p(st["c"]), case["m"],
                                  case["n"], case["k"], case["group"], None))
    return [st["c"]]


def _own_norm(st):
    L, check = _library()
    case, q, k, qo, ko = st["case"], st["q"], st["k"], st["qo"], st["ko"]
    check(L.vmlm_hip_qk_norm_rope(
        _p(qo), qo.stride(0), _p(ko), ko.stride(0), _p(q), q.stride(0), _p(k), k.stride(0),
        _p(st["gq"]), _p(st["gk"]), _p(st["pos"]), case["rows"], case["heads"], case["kv"],
        case["hd"], EPS, THETA, None))
    return [qo, ko]


def _own_cache(st):
    (L, check), desc, w = _library(), _descriptor(st), st["case"]["kv"] * st["case"]["hd"]
    first, count, s = _p(st["first"]), _p(st["count"]), st["case"]["s"]
    check(L.vmlm_hip_kv4_append(desc, _p(st["k"]), w, _p(st["v"]), w, first, count, s, None))
    check(L.vmlm_hip_kv4_read(desc, _p(st["ko"]), w, _p(st["vo"]), w, first, count, s, None))
    return [st["ko"], st["vo"]]


def _own_attn(st):
    (L, check), desc, case = _library(), _descriptor(st), st["case"]
    w, wq, pos = case["kv"] * case["hd"], case["heads"] * case["hd"], _p(st["pos"])
    new = (_p(st["k"]), _p(st["v"])) if case["append"] else (None, None)
    check(L.vmlm_hip_attention_decode_kv4(desc, _p(st["q"]), wq, *new, w, pos, _p(st["out"]),
                                          wq, case["heads"], 1 / math.sqrt(case["hd"]), None, 0,
                                          None))
    if not case["append"]:
        return [st["out"]]
    check(L.vmlm_hip_kv4_read(desc, _p(st["ko"]), w, _p(st["vo"]), w, pos, None, 1, None))
    return [st["out"], st["ko"], st["vo"]]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"linear": _own_linear, "norm": _own_norm, "cache": _own_cache,
                "attn": _own_attn}[kind](state)
    if kind == "linear":
        return [_plain_linear(state)]
    if kind == "norm":
        hd = state["case"]["hd"]
        return [_plain_norm(state["q"], state["gq"], state["pos"], hd),
                _plain_norm(state["k"], state["gk"], state["pos"], hd)]
    if kind == "cache":
        _store(state["cache"], state["k"], state["v"], state["first"], state["count"])
        _load(state["cache"], state["ko"], state["vo"], state["first"], state["count"])
        return [state["ko"], state["vo"]]
    return _plain_attn(state)


# ------------------------------------------------------------------ in 64 bits
def _outward(x, way):
    """x (f64) to 8 significant bits, by np.floor or np.ceil."""
    m, e = np.frexp(x)
    return np.ldexp(way(m * 256), e - 8)


def _held(rows):
    """What the 4-bit cache holds of rows (f32): the lowest of 32 values rounded
    down to bf16, a fifteenth of the range up to the highest rounded up to bf16, and
    the nearest of the 16 steps, ties to even. The difference and the quotients
    are f32 by definition, since they decide the codes."""
    x = rows.cpu().numpy().reshape(tuple(rows.shape[:-1]) + (-1, BLOCK))
    low = _outward(x.min(-1).astype(np.float64), np.floor).astype(np.float32)
    step = _outward(((x.max(-1) - low) / np.float32(15)).astype(np.float64), np.ceil)
    low, step = low[..., None], step[..., None].astype(np.float32)
    steps = np.rint((x - low) / np.where(step > 0, step, np.float32(1)))
    held = low.astype(np.float64) + step.astype(np.float64) * np.clip(steps, 0, 15)
    return torch.from_numpy(held.reshape(tuple(rows.shape))).to(DEV)


def _double(codes, meta):
    """Values of unsigned codes [..., hd] and their meta, in f64."""
    ends = meta.view(torch.bfloat16).double()  # little-endian: scale, min
    wide = torch.repeat_interleave(ends.unflatten(-1, (-1, 2)), BLOCK, dim=-2)
    return wide[..., 1] + wide[..., 0] * codes


def _split_bytes(b):
    """The codes 0..15 of bytes, low half first (f64)."""
    out = torch.empty(*b.shape[:-1], 2 * b.shape[-1], device=DEV, dtype=torch.float64)
    for half in range(2):
        out[..., half::2] = ((b.long() // 16 ** half % 16 + 8) % 16).double()
    return out


def _exact_attn(case, st):
    kv, hd, cache = case["kv"], case["hd"], st["cache"]
    out = torch.zeros(case["batch"], case["heads"] * hd, device=DEV, dtype=torch.float64)
    ko, vo = (torch.zeros(*st[x].shape, device=DEV, dtype=torch.float64) for x in "kv")
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        blocks = -(-n // BLOCK)
        vcodes = _split_bytes(cache["v"][b, :, :blocks]).permute(0, 1, 3, 2).reshape(kv, -1, hd)
        k = _double(_split_bytes(cache["k"][b, :, :n]), cache["km"][b, :, :n])
        v = _double(vcodes[:, :n], cache["vm"][b, :, :n])
        if case["append"]:
            ko[b], vo[b] = _held(st["k"][b]), _held(st["v"][b])
            k[:, -1], v[:, -1] = ko[b].view(kv, hd), vo[b].view(kv, hd)
        q = st["q"][b].double().view(kv, -1, hd)
        for h in range(kv):
            p = torch.softmax((q[h] @ k[h].T) / math.sqrt(hd), dim=-1)
            out[b].view(kv, -1, hd)[h] = p @ v[h]
    return [out, ko, vo] if case["append"] else [out]


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "linear":
        w = _split_bytes(st["q"]) - 8
        for i in range(st["s"].shape[1]):
            w[:, i * case["group"]:(i + 1) * case["group"]] *= st["s"][:, i:i + 1].double()
        return [torch.matmul(w, st["a"].double().T.contiguous()).T]
    if kind == "norm":
        got, hd = [], case["hd"]
        turn = torch.exp(torch.arange(hd // 2, device=DEV).double() * (-2 / hd * math.log(THETA)))
        for x, g in ((st["q"], st["gq"]), (st["k"], st["gk"])):
            x = x.double().reshape(case["rows"], -1, hd)
            y = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / hd + EPS) * g.double()
            z = torch.complex(y[..., :hd // 2], y[..., hd // 2:])
            a = st["pos"].double()[:, None] * turn
            z = z * torch.polar(torch.ones_like(a), a)[:, None]
            got.append(torch.cat((z.real, z.imag), dim=-1).reshape(case["rows"], -1))
        return got
    if kind == "cache":
        got = []
        for x in (st["k"], st["v"]):
            y = torch.zeros(*x.shape, device=DEV, dtype=torch.float64)
            for b, n in enumerate(_counts(case)):
                y[b, :n] = _held(x[b, :n])
            got.append(y)
        return got
    return _exact_attn(case, st)
