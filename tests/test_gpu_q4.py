"""Rotary plans and the 4-bit paged cache on the GPU against the formulas in float64 (tests/q4_ref.py)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from powerinfer_x64_amd import runtime as rt
from tests import q4_ref as ref
from tests.gpu_util import device

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def f64(t):
    return t.detach().cpu().double().numpy()


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def normal(rng, *shape, dtype="f32", mul=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * mul).astype(np.float32)).to(DT[dtype]).cuda()


# ---- rotary positions ----------------------------------------------------------------------


def rotation_tol(x, m, dtype):
    """Angle (reduced in f64, 2^-24 turns in f32) and sincospi 4 ulp of 1, products and sum 3 roundings:
    8 * 2^-24 of |x0| + |x1| <= 2 max|x| of the row; then the output's rounding."""
    top = np.abs(x).max(-1, keepdims=True)
    return lambda y: 16 * 2.0 ** -24 * abs(m) * top + np.abs(y) * ref.EPS[dtype] * 1.01 + 2.0 ** -24


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("d,rope_dim", [(64, 64), (128, 128), (256, 64), (128, 34), (80, 80), (66, 2), (256, 256), (72, 16)])
def test_rope_layouts_widths_types(dtype, layout, d, rope_dim):
    dev, rng = device(), np.random.default_rng(d * 1000 + rope_dim)
    plan = rt.RopePlan(dev, rope_dim, base=1e6, layout=layout, scaling="yarn", factor=4.0)
    n, hq, hkv = 37, 5, 3
    q, k = normal(rng, n, hq, d, dtype=dtype), normal(rng, n, hkv, d, dtype=dtype)
    pos = rng.integers(0, 1 << 20, n)
    pos[:4] = [0, 1, 2 ** 31 - 1, 1 << 30]
    qo, ko = rt.rope_apply(dev, plan, q, k, i32(pos))
    for x, y in ((q, qo), (k, ko)):
        want = ref.rotate(f64(x), pos, plan.freqs, plan.mscale, layout)
        assert y.dtype == x.dtype and y.is_contiguous()
        assert (np.abs(f64(y) - want) <= rotation_tol(f64(x), plan.mscale, dtype)(want)).all()
        assert torch.equal(y[..., rope_dim:], x[..., rope_dim:])  # the rest of the head, bit for bit


@pytest.mark.parametrize("dtype,d,rope_dim", [("f16", 128, 128), ("f32", 64, 18), ("bf16", 256, 64)])
@pytest.mark.parametrize("where", ["fused", "head_major", "odd_offset", "in_place", "in_place_fused"])
def test_rope_strides(dtype, d, rope_dim, where):
    """Rows out of fused projections, head-major tensors, unaligned rows, in place: the same bits as contiguous rows
    (each route's own kernel is held to the formula above)."""
    dev, rng = device(), np.random.default_rng(11)
    plan = rt.RopePlan(dev, rope_dim, base=1e4, layout="halves")
    n, hq, hkv = 19, 4, 2
    base = normal(rng, n, hq + 2 * hkv, d, dtype=dtype)
    q, k, pos = base[:, :hq].contiguous(), base[:, hq:hq + hkv].contiguous(), i32(rng.integers(0, 5000, n))
    want = rt.rope_apply(dev, plan, q, k, pos)
    if where == "fused":
        got = rt.rope_apply(dev, plan, base[:, :hq], base[:, hq:hq + hkv], pos)
    elif where == "head_major":
        hm = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k)]
        out = [torch.empty_like(x.transpose(0, 1).contiguous()).transpose(0, 1) for x in (q, k)]
        got = rt.rope_apply(dev, plan, *hm, pos, *out)
        assert got[0] is out[0]
    elif where == "odd_offset":
        odd = []
        for x in (q, k):
            b = torch.zeros(x.numel() + 3, dtype=x.dtype, device="cuda")
            b[3:] = x.reshape(-1)
            odd.append(b[3:].view(x.shape))
        got = rt.rope_apply(dev, plan, *odd, pos)
    elif where == "in_place":
        got = [q.clone(), k.clone()]
        rt.rope_apply(dev, plan, *got, pos, *got)
    else:
        b = base.clone()
        got = [b[:, :hq], b[:, hq:hq + hkv]]
        rt.rope_apply(dev, plan, *got, pos, *got)
        assert torch.equal(b[:, hq + hkv:], base[:, hq + hkv:])
    for a, b in zip(got, want):
        x = f64(a)
        tol = 2.0 ** -24 * 8 + np.abs(x) * ref.EPS[dtype] * 2.02  # either kernel is off by half a step
        assert (np.abs(x - f64(b)) <= tol).all() if where == "odd_offset" else torch.equal(a, b)


def test_rope_without_keys_empty_and_single():
    dev, rng = device(), np.random.default_rng(12)
    plan = rt.RopePlan(dev, 64, base=1e4)
    q = normal(rng, 1, 32, 128, dtype="f16")
    a, none = rt.rope_apply(dev, plan, q, None, i32([77]))
    assert none is None
    want = ref.rotate(f64(q), [77], plan.freqs, 1.0, "halves")
    assert (np.abs(f64(a) - want) <= rotation_tol(f64(q), 1.0, "f16")(want)).all()
    e, _ = rt.rope_apply(dev, plan, q[:0], None, i32([]))
    assert e.shape == (0, 32, 128)
    own = rt.RopePlan(dev, 8, freqs=[1.0, 0.5, 0.25, 0.0], mscale=0.5, layout="pairs")
    a, _ = rt.rope_apply(dev, own, q, None, i32([-9]))
    want = ref.rotate(f64(q), [-9], [1.0, 0.5, 0.25, 0.0], 0.5, "pairs")
    assert (np.abs(f64(a) - want) <= rotation_tol(f64(q), 1.0, "f16")(want)).all()


def test_rope_refusals():
    dev = device()
    plan = rt.RopePlan(dev, 64)
    q = torch.zeros(4, 2, 128, device="cuda")
    pos = i32([0, 1, 2, 3])
    for bad in (lambda: rt.RopePlan(dev, 258), lambda: rt.RopePlan(dev, 63), lambda: rt.RopePlan(dev, 64, layout="x"),
                lambda: rt.RopePlan(dev, 8, freqs=[1.0]), lambda: rt.RopePlan(dev, 4, freqs=[1.0, math.nan]),
                lambda: rt.RopePlan(dev, 64, mscale=math.inf),
                lambda: rt.rope_apply(dev, plan, q.double(), None, pos), lambda: rt.rope_apply(dev, plan, q.cpu(), None, pos),
                lambda: rt.rope_apply(dev, plan, q, None, pos[:3]), lambda: rt.rope_apply(dev, plan, q, None, pos.long()),
                lambda: rt.rope_apply(dev, plan, q, q.half(), pos), lambda: rt.rope_apply(dev, plan, q[..., :32], None, pos),
                lambda: rt.rope_apply(dev, plan, q[..., ::2], None, pos),
                lambda: rt.rope_apply(dev, plan, q, None, pos, q_out=q[:1].expand(4, 2, 128)),
                lambda: rt.rope_apply(dev, plan, q[0], None, pos),
                lambda: rt.rope_apply(dev, plan, q, None, pos, q_out=q.view(2, 4, 128).transpose(0, 1))):
        with pytest.raises((rt.InvalidArg, rt.Unsupported)):
            bad()


# ---- the cache -----------------------------------------------------------------------------


class Cache:
    """A pool whose pages hold seeded records, and the same keys and values in float64."""

    def __init__(self, rng, lens, hkv, d, spare=3, wide=0):
        self.dev, self.hkv, self.d, self.lens = device(), hkv, d, list(lens)
        used = [(n + 15) // 16 for n in lens]
        self.max_pages = max(max(used, default=0), 1) + wide
        self.n_pages = sum(used) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((max(len(lens), 1), self.max_pages), -1, np.int32)
        at = 0
        for i, u in enumerate(used):
            self.table[i, :u] = order[at:at + u]
            at += u
        self.pool = rt.Q4Pool(self.dev, self.n_pages, hkv, d)
        self.pt = torch.from_numpy(self.table).cuda()
        self.k, self.v = [], []
        # every slot of the pool holds something, the largest values among the unused ones
        every = torch.arange(self.n_pages, dtype=torch.int32, device="cuda").view(1, -1)
        junk = [torch.full(s, 0xF0 if t == torch.uint8 else 904.0, dtype=t, device="cuda")
                for t, s in self.pool._record_shapes(16 * self.n_pages)]
        self.pool.write(every, 0, 0, *junk)
        for i, n in enumerate(lens):
            recs, vals = [], []
            for _ in range(2):
                c, s = ref.quantise(rng.standard_normal((n, hkv, d)))
                vals.append(ref.values(c, s))
                recs += [torch.from_numpy(ref.pack(c)).cuda(), torch.from_numpy(s.astype(np.float16)).cuda()]
            self.k.append(vals[0])
            self.v.append(vals[1])
            if n:
                self.pool.write(self.pt, i, 0, *recs)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_records_come_back_bit_for_bit(d):
    rng = np.random.default_rng(d)
    c = Cache(rng, [37, 1, 16, 0], 3, d)
    for i, n in enumerate(c.lens):
        kc, ks, vc, vs = c.pool.read(c.pt, i, 0, n)
        assert np.array_equal(ref.values(ref.unpack(kc.cpu()), f64(ks)), c.k[i])
        assert np.array_equal(ref.values(ref.unpack(vc.cpu()), f64(vs)), c.v[i])
    kc, ks, vc, vs = c.pool.read(c.pt, 0, 5, 20)  # from inside a page to inside another
    assert np.array_equal(ref.values(ref.unpack(kc.cpu()), f64(ks)), c.k[0][5:25])
    before = c.pool.read(c.pt, 0, 0, 37)
    c.pool.write(c.pt, 0, 5, kc, ks, vc, vs)
    assert all(torch.equal(a, b) for a, b in zip(before, c.pool.read(c.pt, 0, 0, 37)))
    # positions without a page: zeros out, nothing in
    kc, ks, vc, vs = c.pool.read(c.pt, 1, 0, 40)
    assert (kc[16:] == 0x88).all() and (ks[16:] == 0).all() and (vc[16:] == 0x88).all() and (vs[16:] == 0).all()
    c.pool.write(c.pt, 1, 16, kc[:24], ks[:24], vc[:24], vs[:24])
    assert all(torch.equal(a, b) for a, b in zip(before, c.pool.read(c.pt, 0, 0, 37)))


def test_write_takes_no_scale_off_the_grid():
    c = Cache(np.random.default_rng(1), [16], 1, 64)
    kc, ks, vc, vs = (t.clone() for t in c.pool.read(c.pt, 0, 0, 16))
    bits = torch.tensor([0x7E00, 0x7C00, 0xFC00, 0xFFFF, 0x7BFF, 0x6311, 0x6320, 0xE320, 0x3C0F, 0x000F, 0x8010, 0x7C01, 0, 0x8000,
                         0x3C10, 0xBC00], dtype=torch.int32).to(torch.int16).view(torch.float16).cuda()
    ks[:, 0, 0] = bits
    c.pool.write(c.pt, 0, 0, kc, ks, vc, vs)
    got = c.pool.read(c.pt, 0, 0, 16)[1][:, 0, 0].view(torch.int16).cpu().numpy().astype(np.uint16)
    assert [hex(x) for x in got] == [hex(x) for x in (0, 0x6310, 0xE310, 0, 0x6310, 0x6310, 0x6310, 0xE310, 0x3C00, 0, 0x8010, 0, 0, 0x8000,
                                                      0x3C10, 0xBC00)]


def check_append(dtype, d, hq, hkv, toks, starts, norm, layout, rope_dim, fused=True, tok_start=True, seed=0, edit=None, plan_on=True):
    rng = np.random.default_rng(seed)
    lens = [s + n for s, n in zip(starts, toks)]
    c = Cache(rng, lens, hkv, d)
    n, tail = sum(toks), 2 if tok_start else 0
    x = normal(rng, n + tail, hq + 2 * hkv, d, dtype=dtype)
    if edit:
        edit(x)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    plan = rt.RopePlan(c.dev, rope_dim, base=1e6, layout=layout, scaling="bands", factor=4.0) if plan_on else None
    qw = kw = None
    if norm:
        qw, kw = (1 + 0.1 * normal(rng, d) for _ in range(2))
    ts = np.concatenate([[0], np.cumsum(toks)])
    q_out = torch.full((n + tail, hq, d), 7.0, dtype=DT[dtype], device="cuda")
    qo, kv, vv = c.pool.append(k, v, c.pt, i32(starts), tok_start=i32(ts) if tok_start else None, plan=plan, q=q, q_norm_w=qw,
                               k_norm_w=kw, eps=1e-6, q_out=q_out, values=True)
    assert qo is q_out
    pos = np.concatenate([np.arange(s, s + t) for s, t in zip(starts, toks)]).astype(np.int64)
    rot = lambda a: ref.rotate(a, pos, plan.freqs, plan.mscale, layout) if plan else a  # noqa: E731
    with np.errstate(invalid="ignore"):
        qn, kn, v64 = f64(q)[:n], f64(k)[:n], f64(v)[:n]
        if norm:
            qn, kn = ref.rms(qn, f64(qw), 1e-6), ref.rms(kn, f64(kw), 1e-6)
        want_q, want_k = rot(qn), rot(kn)
    kc, ks = ref.quantise(want_k)
    vc, vs = ref.quantise(v64)
    if edit is None:
        # norm (f32): sum of D squares, root, two products: (D / 2 + 4) 2^-24 relative at most; rotation as in rope_apply
        tol = rotation_tol(qn, 1.0, dtype)(want_q) + (np.abs(qn).max(-1, keepdims=True) * 2 * (d / 2 + 4) * 2.0 ** -24 if norm else 0)
        assert (np.abs(f64(qo)[:n] - want_q) <= tol).all()
        assert (qo[n:] == 7.0).all()
    at = 0
    for i, t in enumerate(toks):
        got = [g.cpu() for g in c.pool.read(c.pt, i, 0, lens[i])]
        # the tokens that were there before are as they were
        assert np.array_equal(ref.values(ref.unpack(got[0][:starts[i]]), f64(got[1][:starts[i]])), c.k[i][:starts[i]])
        assert np.array_equal(ref.values(ref.unpack(got[2][:starts[i]]), f64(got[3][:starts[i]])), c.v[i][:starts[i]])
        s, e = starts[i], at + t
        assert np.array_equal(f64(got[1][s:]), ks[at:e]) and np.array_equal(ref.unpack(got[0][s:]), kc[at:e])
        assert np.array_equal(f64(got[3][s:]), vs[at:e]) and np.array_equal(ref.unpack(got[2][s:]), vc[at:e])
        at = e
    assert np.array_equal(f64(kv)[:n], ref.values(kc, ks)) and np.array_equal(f64(vv)[:n], ref.values(vc, vs))
    return c


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("d,rope_dim,hq,hkv", [(64, 64, 3, 1), (128, 128, 8, 2), (256, 64, 5, 2), (128, 34, 4, 4), (64, 18, 2, 1)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_ragged(dtype, layout, d, rope_dim, hq, hkv, norm):
    """Chunks that start and end inside pages, an empty one, one token, more than a page; codes, scales, values and
    every earlier token exact."""
    check_append(dtype, d, hq, hkv, [5, 0, 1, 40, 16, 17], [3, 9, 0, 13, 16, 30], norm, layout, rope_dim, seed=d + rope_dim)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fused", [True, False])
def test_append_one_token_a_sequence(dtype, fused):
    check_append(dtype, 128, 8, 2, [1] * 70, [int(x) for x in np.random.default_rng(1).integers(0, 60, 70)], True, "halves", 128,
                 fused=fused, tok_start=False)


def test_append_many_rows_and_sequences():
    """Over 1024 rows (several tokens a workgroup) of over 64 sequences (two-level search)."""
    rng = np.random.default_rng(2)
    toks = [int(x) for x in rng.integers(0, 30, 150)]
    check_append("bf16", 64, 2, 1, toks, [int(x) for x in rng.integers(0, 40, 150)], False, "halves", 64)


def test_append_without_plan_or_queries():
    check_append("f16", 128, 2, 1, [20], [7], False, "halves", 128, plan_on=False)
    rng = np.random.default_rng(4)
    c = Cache(rng, [9], 2, 64)
    k, v = normal(rng, 9, 2, 64), normal(rng, 9, 2, 64)
    assert c.pool.append(k, v, c.pt, i32([0]), tok_start=i32([0, 9])) is None
    kc, ks, vc, vs = c.pool.read(c.pt, 0, 0, 9)
    for x, codes, s in ((k, kc, ks), (v, vc, vs)):
        wc, ws = ref.quantise(f64(x))
        assert np.array_equal(ref.unpack(codes.cpu()), wc) and np.array_equal(f64(s), ws)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_append_values_at_the_borders(dtype):
    """Ties of magnitude, quotients of k + 1/2, groups of zeros, tiny and huge groups, NaN and infinities."""
    def edit(x):
        v, k = x[:, 3], x[:, 2]
        for y in (k, v):
            y[0] = 0
            y[1] = (torch.arange(128, device="cuda") % 17 - 8) * 0.25  # +2 and -2, on the grid
            y[2] = (torch.arange(128, device="cuda") % 16) * 0.125 - 0.9375  # halves of steps
            y[2, ::32] = -2.0
            y[3] *= 2.0 ** -14
            y[4] *= 2.0 ** -20
            y[5] *= 2.0 ** -22
            y[6] *= 3000.0
            y[7, 5], y[7, 40], y[7, 70], y[7, 71] = math.nan, math.inf, -math.inf, math.nan
            y[8] = math.nan
            y[9] = -1.0
            y[10] = 60000.0
    check_append(dtype, 128, 2, 1, [16], [0], False, "halves", 128, edit=edit, plan_on=False)


def test_append_tables_are_not_trusted():
    """Positions past the row, page ids outside the pool, negative starts, ranges that do not fit: the rest is stored."""
    rng = np.random.default_rng(6)
    c = Cache(rng, [32, 32], 1, 64, spare=2)
    whole = torch.arange(c.n_pages, dtype=torch.int32, device="cuda").view(1, -1)
    before = [t.clone() for t in c.pool.read(whole, 0, 0, 16 * c.n_pages)]
    k = normal(rng, 20, 1, 64)
    plan = rt.RopePlan(c.dev, 64)
    for table, start, ts in ((np.array([[c.n_pages, -1], [2 ** 31 - 1, -2 ** 31]]), [0, 5], [0, 10, 20]),
                             (c.table, [32, 2 ** 31 - 1], [0, 10, 20]),
                             (c.table, [0, 0], [20, 10, 0]), (c.table, [0, 0], [25, 30, 40]), (c.table, [0, 0], [-5, -2, -1])):
        q = c.pool.append(k, k, i32(table), i32(start), tok_start=i32(ts), plan=plan, q=k)
        assert q.shape == k.shape
        assert all(torch.equal(a, b) for a, b in zip(before, c.pool.read(whole, 0, 0, 16 * c.n_pages)))
    c.pool.append(k, k, c.pt, i32([-7, 0]), tok_start=i32([-3, 5, 5]))  # rows 0 .. 4 of sequence 0, from position 0
    got = c.pool.read(c.pt, 0, 0, 32)
    wc, ws = ref.quantise(f64(k)[:5])
    assert np.array_equal(ref.unpack(got[0][:5].cpu()), wc) and np.array_equal(f64(got[1][:5]), ws)
    assert np.array_equal(ref.values(ref.unpack(got[0][5:].cpu()), f64(got[1][5:])), c.k[0][5:])


# ---- attention -----------------------------------------------------------------------------


def check_decode(dtype, d, hq, hkv, lens, mode=0, gate=False, seed=0, scale=None, mul=1.0, wide=0, max_ctx=None, bad=(), spare=3):
    rng = np.random.default_rng(seed)
    c = Cache(rng, lens, hkv, d, wide=wide, spare=spare)
    q = normal(rng, len(lens), hq, d, dtype=dtype, mul=mul)
    gt = normal(rng, len(lens), hq, d, dtype=dtype) if gate else None
    masks = [np.zeros(n, bool) for n in lens]
    table = c.table.copy()
    for s, page, what in bad:
        table[s, page] = what
        masks[s][16 * page:16 * page + 16] = True
    out = rt.q4_attn_decode(c.dev, q, c.pool, i32(table), i32(lens), gqa_mode=mode, scale=scale, gate=gt, max_ctx=max_ctx)
    assert out.dtype == q.dtype
    sc = 1 / math.sqrt(d) if scale is None else scale
    kv_of, got = ref.head_map(hq, hkv, mode), f64(out)
    for i, n in enumerate(lens):
        q64 = f64(q)[i:i + 1]
        want = ref.attend(q64, c.k[i], c.v[i], [n - 1], kv_of, sc, f64(gt)[i:i + 1] if gate else None, masks[i])
        assert np.isfinite(got[i]).all()
        err, tol = np.abs(got[i:i + 1] - want), ref.attend_tol(q64, c.k[i], c.v[i], want, sc, dtype)
        assert (err <= tol).all(), (i, n, float((err / tol).max()))
        if n == 0 or masks[i].all():
            assert (got[i] == 0).all()
    return c, q, out


LENS = [1, 0, 15, 16, 17, 31, 32, 33, 64, 100, 300, 1000]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,hq,hkv", [(64, 12, 4), (128, 32, 8), (256, 16, 2), (128, 4, 4), (256, 3, 1)])
def test_decode(dtype, d, hq, hkv):
    check_decode(dtype, d, hq, hkv, LENS, seed=d + hq)


@pytest.mark.parametrize("dtype,d,hq,hkv,mode", [("f16", 128, 32, 8, 1), ("f32", 64, 21, 3, 1), ("bf16", 128, 7, 3, 0),
                                                 ("f16", 64, 71, 1, 1), ("bf16", 256, 40, 2, 0), ("f32", 256, 33, 1, 0),
                                                 ("f16", 128, 2, 5, 0), ("f32", 128, 70, 2, 1)])
def test_decode_head_maps(dtype, d, hq, hkv, mode):
    """Grouped and modulo maps, head counts that do not divide, more than one block of 16 heads, fewer heads than KV heads."""
    check_decode(dtype, d, hq, hkv, [1, 40, 0, 700], mode=mode, gate=True, seed=hq)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_long_splits(dtype, d):
    """Long contexts beside short ones: segments over many workgroups' ranges, joined by the merge."""
    check_decode(dtype, d, 8, 2, [9000, 3, 0, 5001, 4096, 16], gate=True, seed=d)


@pytest.mark.parametrize("lens,wide", [([5], 0), ([5], 500), ([0], 0), ([0, 0, 0], 300), ([257] * 40, 0), ([200, 0, 16] * 30, 200)])
def test_decode_small_launches_and_wide_tables(lens, wide):
    check_decode("f16", 128, 8, 2, lens, wide=wide)
    check_decode("f16", 128, 8, 2, lens, wide=wide, max_ctx=max(max(lens), 1))


def test_decode_max_ctx_cuts_at_a_page():
    c, q, out = check_decode("f32", 64, 4, 2, [100, 40])
    cut = rt.q4_attn_decode(c.dev, q, c.pool, c.pt, i32([100, 40]), max_ctx=50)  # 64 tokens are left of the first
    same = rt.q4_attn_decode(c.dev, q, c.pool, c.pt, i32([64, 40]))
    assert torch.allclose(cut, same, rtol=0, atol=1e-5) and not torch.allclose(cut[0], out[0], rtol=0, atol=1e-3)
    over = rt.q4_attn_decode(c.dev, q, c.pool, c.pt, i32([2 ** 31 - 1, -5]))  # clamped to the row, to nothing
    assert torch.isfinite(over).all() and (over[1] == 0).all()


def test_decode_bad_pages_hold_no_tokens():
    check_decode("f16", 128, 8, 2, [100, 40, 17, 33], bad=[(0, 0, -1), (0, 6, 1 << 30), (1, 1, 99999), (2, 0, -7), (2, 1, -7), (3, 2, 10 ** 6)])
    check_decode("f32", 256, 2, 1, [2000], bad=[(0, p, -1) for p in range(0, 125, 2)])
    check_decode("bf16", 64, 2, 1, [3000], bad=[(0, p, -1) for p in range(188)])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_decode_scales(dtype, scale):
    check_decode(dtype, 64, 4, 2, [300, 5], scale=scale)


@pytest.mark.parametrize("dtype,mul", [("bf16", 1e6), ("bf16", 1e-8), ("f32", 1e9), ("f32", 1e-9), ("f16", 1e3)])
def test_decode_query_magnitudes(dtype, mul):
    """Queries whose exponents f16 does not hold, and scores far apart: the scale brings them back to about 8."""
    check_decode(dtype, 128, 4, 2, [500, 3], mul=mul, scale=1 / (mul * math.sqrt(128)))


def test_decode_peaked_rows():
    """Scores hundreds apart: one key wins, the running maximum moves again and again."""
    check_decode("f32", 128, 4, 2, [700, 5], scale=3.0)
    check_decode("f16", 128, 4, 2, [700, 5], scale=3.0)


def test_nan_row_stays_alone():
    rng = np.random.default_rng(8)
    c = Cache(rng, [50, 50], 1, 128)
    q = normal(rng, 2, 4, 128, dtype="f16")
    clean = rt.q4_attn_decode(c.dev, q, c.pool, c.pt, i32([50, 50]))
    q[0, 1, 3] = math.nan
    out = rt.q4_attn_decode(c.dev, q, c.pool, c.pt, i32([50, 50]))
    assert torch.isnan(out[0, 1]).all()
    assert torch.equal(out[0, [0, 2, 3]], clean[0, [0, 2, 3]]) and torch.equal(out[1], clean[1])


def check_prefill(dtype, d, hq, hkv, toks, starts, mode=0, gate=False, seed=0, max_tok=None, tail=3, bad=(), wide=0):
    rng = np.random.default_rng(seed)
    lens = [s + n for s, n in zip(starts, toks)]
    c = Cache(rng, lens, hkv, d, wide=wide)
    n = sum(toks)
    q = normal(rng, n + tail, hq, d, dtype=dtype)
    gt = normal(rng, n + tail, hq, d, dtype=dtype) if gate else None
    out = torch.full_like(q, 5.0)
    masks = [np.zeros(x, bool) for x in lens]
    table = c.table.copy()
    for s, page, what in bad:
        table[s, page] = what
        masks[s][16 * page:16 * page + 16] = True
    ts = np.concatenate([[0], np.cumsum(toks)])
    rt.q4_attn_prefill(c.dev, q, c.pool, i32(table), i32(starts), i32(ts), max_tok=max_tok, gqa_mode=mode, gate=gt, out=out)
    kv_of, sc, got = ref.head_map(hq, hkv, mode), 1 / math.sqrt(d), f64(out)
    for i, t in enumerate(toks):
        rows = slice(ts[i], ts[i] + (t if max_tok is None else min(t, max_tok)))
        m = rows.stop - rows.start
        q64 = f64(q)[rows]
        pos = np.arange(starts[i], starts[i] + m)
        want = ref.attend(q64, c.k[i], c.v[i], pos, kv_of, sc, f64(gt)[rows] if gate else None, masks[i])
        if m:
            err, tol = np.abs(got[rows] - want), ref.attend_tol(q64, c.k[i], c.v[i], want, sc, dtype)
            assert (err <= tol).all(), (i, t, float((err / tol).max()), np.argwhere(err > tol)[:4].tolist())
        assert (got[rows.stop:ts[i + 1]] == 5.0).all()  # past max_tok: as they were
    assert (out[n:] == 5.0).all()
    return c


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,hq,hkv", [(64, 12, 4), (128, 8, 2), (256, 8, 1), (128, 3, 3)])
def test_prefill_ragged(dtype, d, hq, hkv):
    check_prefill(dtype, d, hq, hkv, [1, 0, 5, 16, 33], [0, 40, 100, 13, 600], mode=1, gate=d == 128, seed=d)


@pytest.mark.parametrize("dtype,d,hq,hkv", [("f16", 128, 8, 2), ("bf16", 128, 4, 4), ("f32", 64, 6, 2), ("f16", 256, 4, 1), ("f32", 256, 2, 1),
                                            ("bf16", 64, 14, 2), ("f32", 128, 5, 1)])
def test_prefill_prompts(dtype, d, hq, hkv):
    """Fresh prompts and chunks of hundreds of rows, odd lengths, the causal edge inside every tile."""
    check_prefill(dtype, d, hq, hkv, [257, 130, 64], [0, 5, 777], seed=hq)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_prefill_max_tok_bad_pages_wide_table(dtype):
    check_prefill(dtype, 128, 4, 2, [7, 3, 12], [20, 0, 300], max_tok=6, seed=1)
    check_prefill(dtype, 64, 4, 2, [40, 20], [60, 3], bad=[(0, 0, -1), (0, 3, 99999), (1, 0, -1), (1, 1, -1)], seed=2, wide=9)
    check_prefill(dtype, 128, 4, 2, [140], [60], bad=[(0, 0, -1), (0, 5, 99999), (0, 12, -1)], seed=3, wide=100)


def test_prefill_head_maps():
    check_prefill("f16", 128, 7, 3, [9, 90], [100, 3], mode=0, gate=True)
    check_prefill("f16", 64, 71, 1, [3, 40], [100, 3], mode=1)
    check_prefill("bf16", 128, 2, 5, [9, 70], [100, 3], mode=0)


def test_prefill_tables_are_not_trusted():
    rng = np.random.default_rng(9)
    c = Cache(rng, [64, 64], 2, 128)
    q = normal(rng, 24, 4, 128, dtype="f16")
    for ts, start in (([0, 30, 60], [0, 0]), ([20, 10, 0], [0, 0]), ([-9, 12, 12], [-5, 3]), ([0, 12, 24], [2 ** 31 - 1, 60]),
                      ([2 ** 31 - 1, -2 ** 31, 7], [5, 5])):
        out = rt.q4_attn_prefill(c.dev, q, c.pool, c.pt, i32(start), i32(ts), out=torch.zeros_like(q))
        assert torch.isfinite(out).all()


def test_long_cache_offsets():
    """Pages whose bytes lie past 2^32: the cache's last pages and its first ones give the same rows."""
    dev, rng = device(), np.random.default_rng(10)
    d, hkv, n = 256, 8, 70
    n_pages = (1 << 32) // (18 * d * hkv) + 40
    pool = rt.Q4Pool(dev, n_pages, hkv, d)
    assert pool.nbytes > 1 << 32
    recs = []
    for _ in range(2):
        c, s = ref.quantise(rng.standard_normal((n, hkv, d)))
        recs += [torch.from_numpy(ref.pack(c)).cuda(), torch.from_numpy(s.astype(np.float16)).cuda()]
    table = i32([[n_pages - 1 - i for i in range(5)], [i for i in range(5)]])
    q = normal(rng, 1, 16, d, dtype="bf16")
    k = normal(rng, 3, hkv, d, dtype="bf16")
    for s in (0, 1):
        pool.write(table, s, 0, *recs)
    pool.append(k, k, table, i32([0]), tok_start=i32([0, 3]))
    pool.append(k, k, table[1:], i32([0]), tok_start=i32([0, 3]))
    assert all(torch.equal(a, b) for a, b in zip(pool.read(table, 0, 0, n), pool.read(table, 1, 0, n)))
    out = rt.q4_attn_decode(dev, q.expand(2, 16, d).contiguous(), pool, table, i32([n, n]))
    assert torch.equal(out[0], out[1]) and out.float().abs().sum() > 0
    rows = normal(rng, 160, 16, d, dtype="bf16")
    big = rt.q4_attn_prefill(dev, torch.cat((rows, rows)), pool, table.repeat(1, 2), i32([0, 0]), i32([0, 160, 320]), 160)
    assert torch.equal(big[:160], big[160:])
    pool.close()


# ---- how it is called ----------------------------------------------------------------------


def serve(dev, pool, plan, pt, steps, x, prompt, hq, hkv, ws=None):
    """A prompt appended and attended, then one token at a time; every output."""
    n = int(prompt.sum())
    ts = i32(np.concatenate([[0], np.cumsum(prompt)]))
    zero = i32([0] * len(prompt))
    cut = lambda r: (r[:, :hq], r[:, hq:hq + hkv], r[:, hq + hkv:])  # noqa: E731
    q, k, v = cut(x[:n])
    qr, kv, vv = pool.append(k, v, pt, zero, tok_start=ts, plan=plan, q=q, values=True)
    outs = [qr, kv, vv, rt.q4_attn_prefill(dev, qr, pool, pt, zero, ts, int(prompt.max()))]
    pos = torch.from_numpy(prompt.astype(np.int32)).cuda()
    for i in range(steps):
        q, k, v = cut(x[n + i * len(prompt):n + (i + 1) * len(prompt)])
        qr = pool.append(k, v, pt, pos, plan=plan, q=q)
        pos = pos + 1
        outs += [qr, rt.q4_attn_decode(dev, qr, pool, pt, pos)]
    return outs


def test_run_of_the_operators_together():
    """Ragged prompts, then decode steps, against float64 over what the cache holds; the first prompt also by the dense
    prefill over the values that the append gives back."""
    dev, rng = device(), np.random.default_rng(20)
    hq, hkv, d, prompt, steps = 8, 2, 128, np.array([70, 1, 33]), 5
    n, b = int(prompt.sum()), len(prompt)
    plan = rt.RopePlan(dev, d, base=1e6, scaling="ntk", factor=2.0)
    pool = rt.Q4Pool(dev, 24, hkv, d)
    pt = i32(rng.permutation(24).reshape(3, 8))
    x = normal(rng, n + steps * b, hq + 2 * hkv, d, dtype="f16")
    outs = serve(dev, pool, plan, pt, steps, x, prompt, hq, hkv)
    at = np.concatenate([[0], np.cumsum(prompt)])
    held = []
    for s in range(b):
        kc, ks, vc, vs = pool.read(pt, s, 0, int(prompt[s]) + steps)
        held.append((ref.values(ref.unpack(kc.cpu()), f64(ks)), ref.values(ref.unpack(vc.cpu()), f64(vs))))
        m = int(prompt[s])
        raw = f64(x[at[s]:at[s + 1], hq:hq + hkv])
        kq = ref.quantise(ref.rotate(raw, np.arange(m), plan.freqs, plan.mscale, "halves"))
        assert np.array_equal(ref.values(*kq), held[s][0][:m])
        q64 = f64(outs[0][at[s]:at[s + 1]])
        want = ref.attend(q64, held[s][0], held[s][1], np.arange(m), ref.head_map(hq, hkv, 0), d ** -0.5)
        assert (np.abs(f64(outs[3][at[s]:at[s + 1]]) - want) <= ref.attend_tol(q64, *held[s], want, d ** -0.5, "f16")).all()
    dense = rt.attn_prefill(dev, outs[0][:70].unsqueeze(0).contiguous(), outs[1][:70].unsqueeze(0).contiguous(),
                            outs[2][:70].unsqueeze(0).contiguous())[0]
    vm = float(outs[2][:70].abs().max())
    # the dense kernel scales q before it rounds it to f16: 2^-11 of the scores on top of attend_tol's roundings
    smax = float((outs[0][:70].double().abs().amax(-1).max() * outs[1][:70].double().abs().sum(-1).max())) * d ** -0.5
    assert float((dense.double() - outs[3][:70].double()).abs().max()) <= vm * (2 * smax * 2.0 ** -11 + 4 * 2.0 ** -11)
    for i in range(steps):
        q, o = outs[4 + 2 * i], outs[5 + 2 * i]
        for s in range(b):
            m, q64 = int(prompt[s]) + i, f64(q[s:s + 1])
            want = ref.attend(q64, held[s][0], held[s][1], [m], ref.head_map(hq, hkv, 0), d ** -0.5)
            assert (np.abs(f64(o[s:s + 1]) - want) <= ref.attend_tol(q64, *held[s], want, d ** -0.5, "f16")).all()


def test_the_same_call_gives_the_same_bits():
    dev, rng = device(), np.random.default_rng(21)
    plan, prompt = rt.RopePlan(dev, 128, base=1e6), np.array([300, 9])
    pt = i32(rng.permutation(48).reshape(2, 24))
    x = normal(rng, int(prompt.sum()) + 4, 12, 128, dtype="bf16")
    runs = []
    for _ in range(3):
        pool = rt.Q4Pool(dev, 48, 2, 128)
        runs.append(serve(dev, pool, plan, pt, 2, x, prompt, 8, 2))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def _capture(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(gr, stream=side):
            res = fn()
    torch.cuda.synchronize()
    return gr, res


def test_captured_step_replays():
    """A decode step and a chunk captured, replayed several times with other inputs and eager work between; two captured
    graphs and eager calls have workspaces of their own."""
    dev, rng = device(), np.random.default_rng(22)
    hq, hkv, d, b = 8, 2, 128, 5
    lens = [3000, 1, 700, 64, 33]
    c = Cache(rng, [n + 8 for n in lens], hkv, d)
    plan = rt.RopePlan(dev, d)
    x = normal(rng, b, hq + 2 * hkv, d, dtype="f16")
    pos = i32(lens)
    ts = i32(np.arange(b + 1))
    cut = lambda r: (r[:, :hq], r[:, hq:hq + hkv], r[:, hq + hkv:])  # noqa: E731

    def step():
        q, k, v = cut(x)
        qr = c.pool.append(k, v, c.pt, pos, plan=plan, q=q)
        return rt.q4_attn_decode(dev, qr, c.pool, c.pt, pos + 1), rt.rope_apply(dev, plan, q, k, pos)[1]

    def chunk():
        return rt.q4_attn_prefill(dev, x[:, :hq].contiguous(), c.pool, c.pt, pos, ts, 1)

    step(), chunk()
    g1, r1 = _capture(step)
    g2, r2 = _capture(chunk)
    for rep in range(4):
        x.copy_(normal(rng, b, hq + 2 * hkv, d, dtype="f16"))
        pos.copy_(i32([n + rep for n in lens]))
        torch.cuda.synchronize()
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*r1, r2)]
        want = [*step(), chunk()]
        torch.cuda.synchronize()
        for a, w in zip(got, want):
            assert torch.equal(a, w), rep


def test_streams_and_callers_workspace():
    """The same calls on two streams at once, each with its own workspace, and one given by the caller."""
    dev, rng = device(), np.random.default_rng(23)
    c = Cache(rng, [5000, 300], 2, 128)
    q = normal(rng, 2, 8, 128, dtype="f16")
    ctx = i32([5000, 300])
    want = rt.q4_attn_decode(dev, q, c.pool, c.pt, ctx)
    need = ctypes.c_size_t()
    dev.check(dev.lib.pi_q4_attn_ws_bytes(dev.h, c.pool.p, rt.F16, 2, 2, 1, c.max_pages, 0, 8, 0, ctypes.byref(need)))
    assert need.value > 0
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                ws = torch.full((need.value,), 255, dtype=torch.uint8, device="cuda")
                outs.append(rt.q4_attn_decode(dev, q, c.pool, c.pt, ctx, ws=ws))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    with pytest.raises(rt.InvalidArg, match="workspace"):
        rt.q4_attn_decode(dev, q, c.pool, c.pt, ctx, ws=torch.empty(need.value - 1, dtype=torch.uint8, device="cuda"))


def test_refusals():
    dev = device()
    pool = rt.Q4Pool(dev, 8, 2, 128)
    pt, pos, ts = i32([[0, 1], [2, 3]]), i32([0, 0]), i32([0, 2, 4])
    kv = torch.zeros(4, 2, 128, device="cuda", dtype=torch.float16)
    q = torch.zeros(4, 4, 128, device="cuda", dtype=torch.float16)
    dec = lambda **kw: rt.q4_attn_decode(dev, **{**dict(q=q[:2], pool=pool, page_table=pt, ctx_len=i32([3, 4])), **kw})  # noqa: E731
    pre = lambda **kw: rt.q4_attn_prefill(dev, **{**dict(q=q, pool=pool, page_table=pt, start_pos=pos, tok_start=ts), **kw})  # noqa: E731
    app = lambda **kw: pool.append(**{**dict(k=kv, v=kv, page_table=pt, start_pos=pos, tok_start=ts, q=q), **kw})  # noqa: E731
    dec(), pre(), app()
    buf = torch.zeros(4 * 4 * 128 + 1, device="cuda", dtype=torch.float16)
    long = i32(np.zeros(5000))
    for bad in (lambda: rt.Q4Pool(dev, 0, 2, 128), lambda: rt.Q4Pool(dev, 8, 0, 128), lambda: rt.Q4Pool(dev, 8, 2, 96),
                lambda: rt.Q4Pool(dev, 8, 2, 128, page_tokens=32),
                lambda: dec(q=q[:2].double()), lambda: dec(q=q[:2, :, :64]), lambda: dec(q=q[:2].transpose(0, 1)),
                lambda: dec(ctx_len=i32([3])), lambda: dec(page_table=pt[:1]), lambda: dec(page_table=pt.long()),
                lambda: dec(gqa_mode=2), lambda: dec(q=q[:2, :3].contiguous(), gqa_mode=1), lambda: dec(gate=q[:2].float()),
                lambda: dec(out=q[:2].float()), lambda: dec(max_ctx=-1), lambda: dec(q=q[:2].cpu()),
                lambda: dec(q=buf[1:].view(4, 4, 128)[:2]), lambda: dec(ws="x"),
                lambda: rt.q4_attn_decode(dev, torch.zeros(5000, 4, 128, device="cuda"), pool, i32(np.zeros((5000, 2))), long),
                lambda: pre(tok_start=ts[:2]), lambda: pre(tok_start=ts.long()), lambda: pre(max_tok=-1), lambda: pre(start_pos=pos.float()),
                lambda: pre(q=buf[1:].view(4, 4, 128)),
                lambda: app(k=kv.float()), lambda: app(v=kv[:3]), lambda: app(q=q.float()), lambda: app(q_out=q), lambda: app(eps=-1.0),
                lambda: app(eps=math.nan), lambda: app(tok_start=None), lambda: app(tok_start=ts[:2]), lambda: app(plan=rt.RopePlan(dev, 256)),
                lambda: app(q_norm_w=torch.zeros(64, device="cuda")), lambda: app(k=kv[..., :64], v=kv[..., :64]),
                lambda: app(q_out=q[:1].expand(4, 4, 128)), lambda: app(start_pos=long, tok_start=i32(np.zeros(5001)), page_table=i32(np.zeros((5000, 1)))),
                lambda: pool.read(pt, 2, 0, 1), lambda: pool.read(pt, 0, -1, 1), lambda: pool.read(pt, 0, 0, -1),
                lambda: pool.write(pt, 0, 0, *pool.read(pt, 0, 0, 2)[:3], torch.zeros(1, device="cuda"))):
        with pytest.raises((rt.InvalidArg, rt.Unsupported)):
            bad()
    empty = rt.q4_attn_decode(dev, q[:0], pool, pt[:0], i32([]))
    assert empty.shape == (0, 4, 128)
    assert rt.q4_attn_prefill(dev, q[:0], pool, pt, pos, i32([0, 0, 0])).shape == (0, 4, 128)
    assert all(t.shape[0] == 0 for t in pool.read(pt, 0, 0, 0))


# ---- choices of the launch, and what it refuses ------------------------------------------------


@pytest.mark.parametrize("dtype,d,hq,hkv,n,top", [("f16", 128, 8, 2, 140, 1500), ("f32", 64, 4, 4, 70, 2000), ("bf16", 256, 16, 16, 24, 1500),
                                                  ("f16", 64, 32, 32, 24, 4000), ("bf16", 256, 8, 8, 25, 1980), ("f16", 64, 8, 8, 32, 6500)])
def test_decode_many_segments(dtype, d, hq, hkv, n, top):
    """A segment for every CU: whole ones up to a size, items of half the pages past it."""
    lens = np.random.default_rng(n).integers(0, top + 1, n).tolist()
    lens[3], lens[-1] = top, 0
    check_decode(dtype, d, hq, hkv, lens, seed=n)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prefill_many_splits(dtype, d):
    """Few row blocks over long histories: up to 32 key splits, some of them empty, joined by the merge."""
    check_prefill(dtype, d, 8, 2, [40], [9000], seed=d)
    check_prefill(dtype, d, 8, 2, [3, 0, 70], [9000, 5, 1], gate=True, seed=d + 1)


def test_prefill_many_sequences_merge():
    """More sequences than the lanes of a row: the merge finds each row's."""
    rng = np.random.default_rng(31)
    toks = rng.integers(0, 20, 100)
    toks[50] = 20
    check_prefill("f16", 64, 4, 1, toks.tolist(), rng.integers(0, 1200, 100).tolist(), seed=31, max_tok=20)


def test_closed_plans_shared_outputs_and_sizes_are_refused():
    dev = device()
    pool = rt.Q4Pool(dev, 8, 2, 128)
    pt = i32([[0, 1], [2, 3]])
    kv = torch.zeros(2, 2, 128, device="cuda", dtype=torch.float16)
    q = torch.zeros(2, 4, 128, device="cuda", dtype=torch.float16)
    gate = torch.zeros_like(q)
    plan = rt.RopePlan(dev, 128)
    plan.close()
    with pytest.raises(rt.InvalidArg, match="closed"):
        pool.append(kv, kv, pt, i32([0, 0]), plan=plan)
    with pytest.raises(rt.InvalidArg, match="closed"):
        rt.rope_apply(dev, plan, q, None, i32([0, 0]))
    for kw in (dict(out=q), dict(gate=gate, out=gate)):
        with pytest.raises(rt.InvalidArg, match="another tensor"):
            rt.q4_attn_decode(dev, q, pool, pt, i32([1, 1]), **kw)
        with pytest.raises(rt.InvalidArg, match="another tensor"):
            rt.q4_attn_prefill(dev, q, pool, pt, i32([0, 0]), i32([0, 1, 2]), **kw)
    with pytest.raises(rt.InvalidArg):
        rt.Q4Pool(dev, 1, 1 << 17, 64)
    plan, p, unsupported = rt.RopePlan(dev, 64), q.data_ptr(), 5  # PI_ERR_UNSUPPORTED
    size = lambda n, d, h: dev.lib.pi_rope_apply(dev.h, plan.p, rt.F16, n, d, p, p, h * d, d, h, p, h * d, d, None, 0, 0, 0, None, 0, 0,  # noqa: E731
                                                 dev.stream())
    assert [size(1 << 24, 64, 1), size(1, 65536, 16385)] == [unsupported] * 2
    rows = (1 << 24, i32([0, 1]).data_ptr(), i32([0]).data_ptr(), 1, pt.data_ptr(), 2)
    assert dev.lib.pi_q4_append(dev.h, pool.p, None, rt.F16, *rows, None, 0, 0, 0, None, 0, 0, p, 256, 128, p, 256, 128, None, None, 0.0,
                                None, None, dev.stream()) == unsupported
    need = ctypes.c_size_t()
    assert dev.lib.pi_q4_attn_ws_bytes(dev.h, pool.p, rt.F16, 1 << 30, 4096, 1 << 30, 4, 0, 8, 0, ctypes.byref(need)) == unsupported


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("d,rope_dim", [(67, 22), (20, 20), (13, 6), (7, 2), (128, 34), (250, 250)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rope_odd_widths_between_guards(dtype, layout, d, rope_dim, in_place):
    """Chunks that end before their eighth channel, rows at odd offsets: nothing beside the rows is written."""
    dev, rng = device(), np.random.default_rng(d + rope_dim)
    plan = rt.RopePlan(dev, rope_dim, base=1e4, layout=layout)
    n, h, gap = 9, 3, 5
    src = normal(rng, n * h * (d + gap) + 1, dtype=dtype)
    dst = src.clone() if in_place else torch.full_like(src, 9.0)
    rows = lambda t: t[1:].view(n, h, d + gap)[..., :d]  # noqa: E731
    pos = rng.integers(0, 5000, n)
    rt.rope_apply(dev, plan, rows(dst if in_place else src), None, i32(pos), rows(dst))
    want = ref.rotate(f64(rows(src)), pos, plan.freqs, 1.0, layout)
    assert (np.abs(f64(rows(dst)) - want) <= rotation_tol(f64(rows(src)), 1.0, dtype)(want)).all()
    assert torch.equal(rows(dst)[..., rope_dim:], rows(src)[..., rope_dim:])
    between = lambda t: t[1:].view(n, h, d + gap)[..., d:]  # noqa: E731
    assert dst[0] == (src[0] if in_place else 9.0)
    assert torch.equal(between(dst), between(src)) if in_place else (between(dst) == 9.0).all()
