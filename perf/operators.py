"""Rotary positions and the 4-bit paged KV cache, as operators that can be timed and compared.

`run` computes them in plain torch operations, or with `own` through the torch front end
(powerinfer_x64_amd.runtime) as a serving program calls it.  A case is a dict of plain values:

  kind "rope"     rope_apply: q and k rows, cut out of a fused projection's rows, rotated at their
                  positions by a plan (layout, rotary part of the head, long-context scaling)
  kind "append"   Q4Pool.append: new tokens of a ragged batch normed, rotated, quantised into their
                  sequences' pages; the rotated q and the values that the cache now stands for come back
  kind "decode"   q4_attn_decode: one token a sequence over its 4-bit cache ("new": the token's
                  keys and values are appended first, as a serving step does)
  kind "prefill"  q4_attn_prefill: a chunk of tokens a sequence over its 4-bit cache, causal

The cache: groups of 32 channels of a token's key or value head.  m is the group's value of largest
magnitude (the positive one of a tie), s = -m / 8 rounded to 7 significant bits (a multiple of
2^-20 below 2^-14, at most 904), code = clamp(rint(x / s), -8, 7) + 8 (8 where s is 0), and the value
s * (code - 8).  Head shapes, contexts and chunk sizes are those of this repository's benchmark
and tests; q, k, v ~ N(0, 1), pages in random order.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
GROUP = 32
S_MAX = 904.0
EPS = 1e-6
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_DEV = None


def _rt():
    from powerinfer_x64_amd import runtime
    return runtime


def _dev():
    """The program's one library handle."""
    global _DEV
    if _DEV is None:
        _DEV = _rt().Device(0)
    return _DEV


# ---- the cases -----------------------------------------------------------------------------

_PLAN = {"layout": "halves", "rope_dim": 128, "base": 1e6, "scaling": "none", "factor": 1.0, "orig": 4096}


def _case(kind, name=None, **kw):
    c = {"kind": kind, "hq": 32, "hkv": 8, "d": 128, "dtype": "f16", "gqa": "modulo", **_PLAN}
    c.update(kw)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # One chat user's next token: the smallest call, all latency.
        _case("rope", "rope_token_f16", n=1, pos_lo=700, pos_hi=700, len_seed=1),
        # A long prompt's rows of a model stretched from 4k to 16k tokens.
        _case("rope", "rope_prompt_bf16_yarn", dtype="bf16", n=4096, pos_lo=0, pos_hi=16383, len_seed=2,
              scaling="yarn", factor=4.0),
        # A full-precision chunk far into a million-token context, a quarter of the head rotated.
        _case("rope", "rope_far_f32_partial", dtype="f32", hq=16, hkv=2, d=256, rope_dim=64, base=1e7, layout="pairs",
              n=1000, pos_lo=900000, pos_hi=1048575, len_seed=3, scaling="bands", factor=8.0, orig=8192),
        # One token of each sequence of a serving batch.
        _case("append", "append_b32_step_f16", batch=32, tok_lo=1, tok_hi=1, pos_lo=1024, pos_hi=32767, len_seed=4,
              norm=False),
        # A whole fresh prompt.
        _case("append", "append_prompt_bf16", dtype="bf16", batch=1, tok_lo=4096, tok_hi=4096, pos_lo=0, pos_hi=0,
              len_seed=5, norm=True, scaling="yarn", factor=4.0),
        # Ragged chunks that start and end inside pages, on a hybrid model's attention layer.
        _case("append", "append_ragged_f32_d256", dtype="f32", hq=16, hkv=2, d=256, rope_dim=64, base=1e7, batch=7,
              tok_lo=1, tok_hi=900, pos_lo=0, pos_hi=9000, len_seed=6, norm=True),
        # One chat user on a small model in full precision: launches and round trips.
        _case("decode", "decode_mha_f32_ctx512", dtype="f32", hkv=32, base=1e4, batch=1, ctx_lo=512, ctx_hi=512,
              len_seed=7, gate=False, new=False),
        # A serving batch of ragged long conversations: bound by the cache's bytes.
        _case("decode", "decode_f16_b32_ragged", batch=32, ctx_lo=1024, ctx_hi=32768, len_seed=8, gate=False, new=False),
        # A serving step at 64k context of a gated hybrid model's attention layer.
        _case("decode", "step_bf16_d256_ctx64k", dtype="bf16", hq=16, hkv=2, d=256, rope_dim=64, base=1e7, batch=8,
              ctx_lo=65536, ctx_hi=65536, len_seed=9, gate=True, new=True, norm=True),
        # A batch whose drafted tokens are checked at once: few rows over long caches.
        _case("prefill", "check_bf16_b8_drafts", dtype="bf16", batch=8, tok_lo=1, tok_hi=8, pos_lo=2000, pos_hi=16000,
              len_seed=10, gate=False, gqa="grouped"),
        # A chunk of a long prompt over what the pages already hold.
        _case("prefill", "chunk_f16_1000_over_8200", batch=1, tok_lo=1000, tok_hi=1000, pos_lo=8200, pos_hi=8200,
              len_seed=11, gate=False),
        # Ragged fresh prompts of a small-head model in full precision.
        _case("prefill", "prompts_f32_d64_ragged", dtype="f32", hq=12, hkv=4, d=64, rope_dim=64, base=1e4, batch=3,
              tok_lo=300, tok_hi=1200, pos_lo=0, pos_hi=0, len_seed=12, gate=False, gqa="grouped"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_heads(rng, d):
    return rng.choice([(16, 2), (8, 2), (16, 4), (5, 1)] if d == 256 else [(32, 8), (32, 32), (8, 4), (12, 4), (16, 2), (21, 3)])


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "decode", "decode", "decode", "prefill", "prefill"])
    d = rng.choice([64, 128, 128, 256])
    hq, hkv = _draw_heads(rng, d)
    scaling = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
    c = _case(kind, hq=hq, hkv=hkv, d=d, dtype=rng.choice(["f16", "bf16", "bf16", "f32"]), gqa=rng.choice(["modulo", "grouped"]),
              layout=rng.choice(["pairs", "halves"]), rope_dim=rng.choice([d, d, d // 2, d // 4 + 2]),
              base=rng.choice([1e4, 1e6, 1e7]), scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
              orig=rng.choice([4096, 8192]), len_seed=rng.randrange(1 << 20))
    if kind == "rope":
        c.update(n=_logint(rng, 1, 8192), pos_lo=_logint(rng, 1, 1 << 20))
        c["pos_hi"] = c["pos_lo"] + _logint(rng, 1, 1 << 17)
        while work(c)["bytes"] > 2.5e8:
            c["n"] = c["n"] * 2 // 3
        return c
    if kind == "decode":
        c.update(batch=_logint(rng, 1, 32), ctx_lo=rng.choice([0, 1, _logint(rng, 16, 8192), _logint(rng, 16, 8192)]),
                 gate=rng.random() < 0.3, new=rng.random() < 0.3, norm=rng.random() < 0.5)
        c["ctx_lo"] = max(c["ctx_lo"], 1 if c["new"] else 0)
        c["ctx_hi"] = max(c["ctx_lo"], 64) * rng.randint(1, 8) + rng.randrange(16)
        while work(c)["bytes"] > 4e8 or c["batch"] * c["ctx_hi"] * hkv * d > 1.1e9:
            c["ctx_hi"] = max(c["ctx_lo"], c["ctx_hi"] // 2)
            c["batch"] = max(1, c["batch"] * 2 // 3)
        return c
    c.update(batch=_logint(rng, 1, 16), tok_lo=rng.choice([0, 1, _logint(rng, 1, 64)]), pos_lo=rng.choice([0, _logint(rng, 1, 8192)]))
    c["tok_hi"] = c["tok_lo"] + _logint(rng, 1, 2048)
    c["pos_hi"] = c["pos_lo"] + rng.choice([0, _logint(rng, 1, 8192)])
    if kind == "append":
        c["norm"] = rng.random() < 0.5
        while work(c)["bytes"] > 1.2e8:
            c["tok_hi"] = max(c["tok_lo"] + 1, c["tok_hi"] * 2 // 3)
            c["batch"] = max(1, c["batch"] * 2 // 3)
        return c
    c["gate"] = rng.random() < 0.3
    most = 2e10 if c["dtype"] == "f32" else 1.2e11
    while work(c)["flops"] > most or c["batch"] * c["tok_hi"] * hq * (c["tok_hi"] + c["pos_hi"]) > 5e8:
        c["tok_hi"] = max(c["tok_lo"] + 1, c["tok_hi"] * 2 // 3)
        c["batch"] = max(1, c["batch"] * 2 // 3)
        c["pos_lo"] = c["pos_lo"] * 2 // 3
        c["pos_hi"] = max(c["pos_lo"], c["pos_hi"] * 2 // 3)
    return c


def _lens(c):
    """(first position, new tokens) of each sequence; a decode's context is their sum.  Only the
    first sequence is never empty."""
    r = random.Random(c["len_seed"])
    if c["kind"] == "decode":
        ctx = [max(r.randint(c["ctx_lo"], c["ctx_hi"]), int(i == 0)) for i in range(c["batch"])]
        return [(max(n - 1, 0), min(n, 1)) for n in ctx]
    return [(r.randint(c["pos_lo"], c["pos_hi"]), max(r.randint(c["tok_lo"], c["tok_hi"]), int(i == 0))) for i in range(c["batch"])]


def _rows(c):
    return sum(n for _, n in _lens(c))


def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    d, hq, hkv = c["d"], c["hq"], c["hkv"]
    if c["kind"] == "rope":  # every row of q and k in and out once
        b = c["n"] * (2 * (hq + hkv) * d * e + 4)
        return {"bytes": b, "flops": 3 * c["n"] * (hq + hkv) * c["rope_dim"]}
    cached = 2 * hkv * (d // 2 + d // GROUP * 2)  # bytes of a token's keys and values in the cache
    lens = _lens(c)
    rows = sum(n for _, n in lens)
    if c["kind"] == "append":  # q in and out, k and v in, their values out, the cache's bytes out
        return {"bytes": rows * (2 * hq * d * e + 2 * hkv * d * (e + 2) + cached), "flops": rows * (3 * hq + 12 * hkv) * d}
    keys = sum(p + n for p, n in lens)
    b = keys * cached + rows * hq * d * e * (3 if c["gate"] else 2)
    if c.get("new"):
        b += rows * (hq * d * e + 2 * hkv * d * e)
    seen = sum(n * p + n * (n + 1) // 2 for p, n in lens)  # (row, key) pairs under the causal mask
    return {"bytes": b, "flops": 4 * d * hq * seen}


# ---- inputs --------------------------------------------------------------------------------

def _freqs(c):
    """Rotary frequencies [rope_dim / 2] in 64 bits and the factor of cos and sin, by the case's scaling."""
    dim, base, fac, orig = c["rope_dim"], c["base"], c["factor"], c["orig"]
    i = torch.arange(dim // 2, dtype=torch.float64)
    if c["scaling"] == "ntk":
        base = base * fac ** (dim / (dim - 2))
    f = base ** (-2.0 * i / dim)
    if c["scaling"] == "linear":
        return f / fac, 1.0
    if c["scaling"] == "yarn":  # pairs that turn over 32 times in the original context keep their speed, under once slow down
        at = lambda turns: dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), dim - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / fac * ramp + f * (1 - ramp), 0.1 * math.log(fac) + 1.0
    if c["scaling"] == "bands":  # wavelengths over the original context slow down, under a quarter of it keep their speed
        turns = orig * f / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / fac * (1 - smooth) + f * smooth, 1.0
    return f, 1.0


def _plan(c):
    rt = _rt()
    return rt.RopePlan(_dev(), c["rope_dim"], base=c["base"], layout=c["layout"], scaling=c["scaling"], factor=c["factor"],
                       orig_ctx=c["orig"])


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _records(g, pages, c):
    """Codes and scales of `pages` pages of keys or values, token by token: [pages, 16, Hkv, D / 2], [.., D / 32]."""
    x = _normal(g, pages, PAGE, c["hkv"], c["d"])
    codes, s = _quantise(x)
    codes = codes.to(torch.uint8).view(pages, PAGE, c["hkv"], c["d"] // 2, 2)
    return codes[..., 0] | (codes[..., 1] << 4), s.to(torch.float16)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, d, hq, hkv = DT[c["dtype"]], c["d"], c["hq"], c["hkv"]
    f, m = _freqs(c)
    st = {"c": c, "f": f.cuda(), "m": m, "plan": _plan(c) if own else None}
    if c["kind"] == "rope":
        r = random.Random(c["len_seed"])
        x = _normal(g, c["n"], hq + 2 * hkv, d).to(dt)  # a fused projection's rows: q, k and v heads
        pos = torch.tensor([r.randint(c["pos_lo"], c["pos_hi"]) for _ in range(c["n"])], dtype=torch.int32)
        st.update(q=x[:, :hq], k=x[:, hq:hq + hkv], pos=pos.cuda())
        return st
    lens = _lens(c)
    rows, batch = sum(n for _, n in lens), len(lens)
    x = _normal(g, rows, hq + 2 * hkv, d).to(dt)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    used = [(p + n + PAGE - 1) // PAGE for p, n in lens]
    max_pages, n_pages = max(max(used), 1), sum(used) + 1
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((batch, max_pages), dtype=torch.int32, device="cuda")
    at = 0
    for s, u in enumerate(used):
        table[s, :u] = order[at:at + u]
        at += u
    st.update(q=q, k=k, v=v, table=table, tok_start=i32(starts), start_pos=i32([p for p, _ in lens]),
              ctx=i32([p + n for p, n in lens]), max_tok=max(n for _, n in lens), gate=None, qw=None, kw=None)
    if c.get("norm"):
        st.update(qw=1 + 0.1 * _normal(g, d), kw=1 + 0.1 * _normal(g, d))
    if c.get("gate"):
        st["gate"] = _normal(g, rows if c["kind"] == "prefill" else batch, hq, d).to(dt)
    if c["kind"] == "decode":  # one row a sequence; a sequence of no tokens has a row too
        st["q"] = _normal(g, batch, hq, d).to(dt)
        if not c["new"]:
            st["k"] = st["v"] = None
    elif c["kind"] == "prefill":
        st["q"] = q.contiguous()
    st["kc"], st["ks"] = _records(g, n_pages, c)
    st["vc"], st["vs"] = _records(g, n_pages, c)
    if own:
        rt = _rt()
        st["mode"] = rt.GROUPED if c["gqa"] == "grouped" else rt.MODULO
        st["pool"] = rt.Q4Pool(_dev(), n_pages, hkv, d)
        if c["kind"] != "append":  # the cache as the sequences' earlier tokens left it
            flat = torch.arange(n_pages, dtype=torch.int32, device="cuda").view(1, -1)
            st["pool"].write(flat, 0, 0, *(st[n].reshape(n_pages * PAGE, hkv, -1) for n in ("kc", "ks", "vc", "vs")))
    return st


# ---- the plain forms -----------------------------------------------------------------------

def _quantise(x):
    """Codes [.., D] and scales [.., D / 32] of x's groups."""
    x = x.reshape(*x.shape[:-1], -1, GROUP)
    hi, lo = x.amax(-1), x.amin(-1)
    s = torch.where(hi >= -lo, hi, lo) / -8
    power = s / torch.where(s == 0, torch.ones_like(s), torch.frexp(s)[0])  # of two, over |s|: an exact quotient
    step = (power / 128).clamp(min=2.0 ** -20)
    s = (torch.round(s / step) * step).clamp(-S_MAX, S_MAX)
    t = torch.where(s[..., None] == 0, torch.zeros_like(x), x / s[..., None])
    return (torch.round(t).clamp(-8, 7) + 8).flatten(-2), s


def _values(codes, s, dtype=torch.float32):
    """The values of codes [.., D] with scales [.., D / 32]."""
    codes = codes.to(dtype) - 8
    return (codes.reshape(*codes.shape[:-1], -1, GROUP) * s.to(dtype)[..., None]).flatten(-2)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def _rotate(x, pos, f, m, layout):
    """x [n, heads, D] in its own precision; the angles in 64 bits."""
    a = (pos.double()[:, None] * f[None, :])[:, None, :]
    cos, sin = (m * torch.cos(a)).to(x.dtype), (m * torch.sin(a)).to(x.dtype)
    half = f.numel()
    part, rest = x[..., :2 * half], x[..., 2 * half:]
    if layout == "pairs":
        x0, x1 = part[..., 0::2], part[..., 1::2]
        y = torch.stack((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1).flatten(-2)
    else:
        x0, x1 = part[..., :half], part[..., half:]
        y = torch.cat((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1)
    return torch.cat((y, rest), -1)


def _norm(x, w):
    if w is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)


def _places(st):
    """Each row's sequence and position."""
    n = int(st["q"].shape[0]) if st["k"] is None else int(st["k"].shape[0])
    row = torch.arange(n, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["tok_start"][1:].contiguous(), row, right=True)
    return seq, row - st["tok_start"][seq] + st["start_pos"][seq]


def _append(st, q):
    c = st["c"]
    seq, pos = _places(st)
    rot = lambda x: _rotate(x, pos, st["f"], st["m"], c["layout"])  # noqa: E731
    # the codes depend on which side of a border a value falls: 64 bits up to there
    kc, ks = _quantise(rot(_norm(st["k"].double(), st["kw"])))
    vc, vs = _quantise(st["v"].double())
    page = st["table"][seq, (pos // PAGE).long()].long()
    slot = (pos % PAGE).long()
    for name, codes, s in (("k", kc, ks), ("v", vc, vs)):
        codes8 = codes.to(torch.uint8)
        st[name + "c"][page, slot] = codes8[..., 0::2] | (codes8[..., 1::2] << 4)
        st[name + "s"][page, slot] = s.to(torch.float16)
    q = rot(_norm(q.float(), st["qw"])).to(q.dtype)
    return q, _values(kc, ks, torch.float64).half(), _values(vc, vs, torch.float64).half()


def _cache(st, which):
    """[batch, Hkv, keys, D] of the sequences' pages."""
    t = st["table"].long()
    codes = _unpack(st[which + "c"][t].flatten(1, 2).transpose(1, 2))
    return _values(codes, st[which + "s"][t].flatten(1, 2).transpose(1, 2))


def _attend(st, q, qpos, live):
    """q [batch, n, Hq, D] at positions qpos [batch, n] (keys up to them, where live) -> the same in 32 bits."""
    c = st["c"]
    b, n, hq, d = q.shape
    hkv, grp = c["hkv"], c["hq"] // c["hkv"]
    grouped = c["gqa"] == "grouped"
    qh = q.float().reshape(b, n, hkv, grp, d) if grouped else q.float().reshape(b, n, grp, hkv, d).transpose(2, 3)
    qh = qh.permute(0, 2, 1, 3, 4).reshape(b, hkv, n * grp, d)
    k, v = _cache(st, "k"), _cache(st, "v")
    s = torch.matmul(qh, k.transpose(-1, -2)).view(b, hkv, n, grp, -1) * (1.0 / math.sqrt(d))
    key = torch.arange(k.shape[2], device="cuda")
    seen = ((key <= qpos[..., None]) & live[..., None])[:, None, :, None, :]
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill(~seen.any(3).any(2)[..., None], 0.0)
    o = torch.matmul(p.view(b, hkv, n * grp, -1), v).view(b, hkv, n, grp, d) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 2, 1, 3, 4)
    return o.reshape(b, n, hq, d) if grouped else o.transpose(2, 3).reshape(b, n, hq, d)


def _plain(st):
    c = st["c"]
    if c["kind"] == "rope":
        return tuple(_rotate(x.float(), st["pos"], st["f"], st["m"], c["layout"]).to(x.dtype) for x in (st["q"], st["k"]))
    if c["kind"] == "append":
        return _append(st, st["q"])
    q = st["q"]
    if c["kind"] == "decode":
        if c["new"]:
            q = _append(st, q)[0]
        o = _attend(st, q[:, None], st["ctx"][:, None] - 1, (st["ctx"] > 0)[:, None])[:, 0]
    else:
        seq, pos = _places({**st, "k": None})
        b, most = st["table"].shape[0], max(st["max_tok"], 1)
        slot = (pos - st["start_pos"][seq]).long()
        padded = torch.zeros((b, most) + q.shape[1:], dtype=q.dtype, device="cuda")
        padded[seq, slot] = q
        qpos = torch.zeros((b, most), dtype=torch.int32, device="cuda")
        qpos[seq, slot] = pos
        live = torch.zeros((b, most), dtype=torch.bool, device="cuda")
        live[seq, slot] = True
        o = _attend(st, padded, qpos, live)[seq, slot]
    if st["gate"] is not None:
        o = o * torch.sigmoid(st["gate"].float())
    return o.to(q.dtype)


# ---- the framework's calls -----------------------------------------------------------------

def _own(st):
    rt, c = _rt(), st["c"]
    if c["kind"] == "rope":
        return rt.rope_apply(_dev(), st["plan"], st["q"], st["k"], st["pos"])
    if c["kind"] == "append":
        return st["pool"].append(st["k"], st["v"], st["table"], st["start_pos"], tok_start=st["tok_start"], plan=st["plan"],
                                 q=st["q"], q_norm_w=st["qw"], k_norm_w=st["kw"], eps=EPS, values=True)
    q = st["q"]
    if c["kind"] == "decode":
        if c["new"]:
            q = st["pool"].append(st["k"], st["v"], st["table"], st["start_pos"], plan=st["plan"], q=q, q_norm_w=st["qw"],
                                  k_norm_w=st["kw"], eps=EPS)
        return rt.q4_attn_decode(_dev(), q, st["pool"], st["table"], st["ctx"], gqa_mode=st["mode"], gate=st["gate"])
    return rt.q4_attn_prefill(_dev(), q, st["pool"], st["table"], st["start_pos"], st["tok_start"], st["max_tok"],
                              gqa_mode=st["mode"], gate=st["gate"])


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits -------------------------------------------------------------

def _exact_turn(x, pos, c):
    """Each rotary pair as one complex number, turned by its angle."""
    dim, half = c["rope_dim"], c["rope_dim"] // 2
    fac, orig, base = c["factor"], c["orig"], c["base"]
    if c["scaling"] == "ntk":
        base *= math.pow(fac, dim / (dim - 2))
    speeds, m = [], 1.0
    for i in range(half):
        w = math.exp(-2.0 * i / dim * math.log(base))
        if c["scaling"] == "linear":
            w /= fac
        elif c["scaling"] == "yarn":
            m = 1.0 + 0.1 * math.log(fac)
            first, last = (dim * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32, 1))
            first, last = max(0, math.floor(first)), min(dim - 1, math.ceil(last))
            r = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            w *= (1 - r) + r / fac
        elif c["scaling"] == "bands":
            r = min(1.0, max(0.0, (orig * w / (2 * math.pi) - 1) / 3))
            w *= r + (1 - r) / fac
        speeds.append(w)
    angle = pos.double()[:, None, None] * torch.tensor(speeds, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full_like(angle, m), angle)
    y = x.double().clone()
    a, b = (slice(0, dim, 2), slice(1, dim, 2)) if c["layout"] == "pairs" else (slice(0, half), slice(half, dim))
    z = torch.complex(y[..., a], y[..., b]) * turn
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_held(x):
    """What the cache holds of x: its groups' scales and whole numbers of them."""
    n = x.unflatten(-1, (-1, GROUP))
    big = n.gather(-1, n.abs().argmax(-1, keepdim=True))
    big = torch.where((n == big.abs()).any(-1, keepdim=True), big.abs(), big)
    raw = -big / 8
    unit = torch.exp2(torch.floor(torch.log2(raw.abs().clamp(min=2.0 ** -14))) - 6).clamp(min=2.0 ** -20)
    s = torch.clamp(unit * torch.round(raw / unit), -S_MAX, S_MAX)
    t = n / torch.where(s == 0, torch.ones_like(s), s)
    low = torch.floor(t)
    up = (t - low > 0.5) | ((t - low == 0.5) & (low.remainder(2) == 1))
    return (s * torch.clamp(low + up, -8, 7)).flatten(-2)


def exact(case, seed):
    c, st = case, prepare(case, seed)
    x64 = lambda x, w: x.double() if w is None else (  # noqa: E731
        x.double() / (x.double().square().sum(-1, keepdim=True) / c["d"] + EPS).sqrt() * w.double())
    if c["kind"] == "rope":
        return _exact_turn(st["q"], st["pos"], c), _exact_turn(st["k"], st["pos"], c)
    lens, d, hq, hkv = _lens(c), c["d"], c["hq"], c["hkv"]
    pos = torch.tensor([p + i for p, n in lens for i in range(n)], dtype=torch.int64, device="cuda")
    if c["kind"] == "append":
        k = _exact_held(_exact_turn(x64(st["k"], st["kw"]), pos, c))
        return _exact_turn(x64(st["q"], st["qw"]), pos, c), k, _exact_held(st["v"].double())
    q = st["q"].double()
    new = None
    if c.get("new"):
        new = (_exact_held(_exact_turn(x64(st["k"], st["kw"]), pos, c)), _exact_held(st["v"].double()))
        q = _exact_turn(x64(st["q"], st["qw"]), pos, c).to(DT[c["dtype"]]).double()  # the step hands q on in its own type
    heads = [h // (hq // hkv) if c["gqa"] == "grouped" else h % hkv for h in range(hq)]
    out, at = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), 0
    for i, (p, n) in enumerate(lens):
        rows = 1 if c["kind"] == "decode" else n
        first, at = at, at + rows
        if n == 0:
            continue
        pages = st["table"][i, :(p + n + PAGE - 1) // PAGE].long()
        kv = []
        for w in ("k", "v"):
            bits = st[w + "c"][pages].flatten(0, 1)[:p + n].double()
            high = torch.floor(bits / 16)
            whole = torch.stack((bits - 16 * high, high), -1).flatten(-2) - 8
            kv.append(whole * st[w + "s"][pages].flatten(0, 1)[:p + n].double().repeat_interleave(GROUP, -1))
        if new is not None:
            kv[0][p], kv[1][p] = new[0][i], new[1][i]
        late = torch.arange(p + n, device="cuda")[None, :] > torch.arange(p, p + n, device="cuda")[:, None]
        for kh in range(hkv):
            mine = [h for h in range(hq) if heads[h] == kh]
            s = torch.matmul(q[first:at, mine].transpose(0, 1), kv[0][:, kh].t().contiguous()) / math.sqrt(d)
            s = s.masked_fill(late, -math.inf)
            out[first:at, mine] = torch.matmul(torch.softmax(s, -1), kv[1][:, kh].contiguous()).transpose(0, 1)
    if st["gate"] is not None:
        out = out / (1 + torch.exp(-st["gate"].double()))
    return out
