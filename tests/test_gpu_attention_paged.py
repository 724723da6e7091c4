"""Attention over a cache in pages (th_build_attention_paged) against the
float64 oracle, every element.

What an element may be off by: a score, a sum of D fp32 products of exact
factors, (D + 8) 2^-24 of the sum of their sizes, and 2^-22 of its own size
through the scale and base-2 exponent; a weight as much relatively, 2^-21 for
its exponential and parts (16 bits' parts: 2^-22); sums over the keys, kept in
32 bits by 4 waves of 32 keys a step, (keys / 128 + 40) 2^-24.  A weighted
mean is off by twice that of the weighted sizes of its values; the result by half a step."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import interpret
from oracle.data import relative
from test_gpu_cache import TYPES, Paged, ints, rows

pytestmark = pytest.mark.gpu

HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _np(t):
    return t.double().cpu().numpy()


def _fill(c, gen, cap):
    """Every page full of rows of N(0, 1), e4m3 ones through the oracle's codes."""
    for name in "kv":
        x = rows(gen, c.dtype, c.pages, c.page, c.KV, c.D, spread=False)
        if c.e4m3:
            codes, scales = interpret.e4m3_rows(_np(x), c.dtype == "f16")
            getattr(c, name).copy_(torch.from_numpy(codes))
            getattr(c, name + "s").copy_(torch.from_numpy(scales))
        else:
            getattr(c, name).copy_(x)


def _attend(c, q, o, lse, lengths, counts=None, **extra):
    import tempest_hip.launch as L
    B, S, H, _ = q.shape
    return L.attention_paged(c.cache, B, H, S, q.data_ptr(), o.data_ptr(), c.table.data_ptr(), lengths.data_ptr(),
                             c.width, lse=lse.data_ptr() if lse is not None else 0,
                             counts=counts.data_ptr() if counts is not None else 0, dtype=c.type, **extra)


def _limits(q, k, v, o, keys, dtype, scale):
    B, S, H, D = q.shape
    group = H // k.shape[2]
    ka, va = np.abs(k).max(1), np.abs(v).max(1)  # over the keys: (B, KV, D)
    sizes = np.einsum("bshd,bhd->bsh", np.abs(q), np.repeat(ka, group, 1)) * scale
    score = sizes * ((D + 8) * 2.0 ** -24 + 2.0 ** -22)
    rel = 2 * (score + 2.0 ** -21 + (keys / 128 + 40) * 2.0 ** -24)
    return rel[..., None] * np.repeat(va, group, 1)[:, None] + HALF_STEP[dtype] * np.abs(o) + 2.0 ** -25, score + 2.0 ** -20


def _check(c, q, o, lse, lengths, counts=None, was=0.0, present=None, k=None, v=None, **masks):
    cap = c.width * c.page
    n = [min(max(int(x), 0), cap) for x in lengths.cpu()]
    m = None if counts is None else counts.cpu().numpy()
    k = c.sequences(cap, "k") if k is None else k
    v = c.sequences(cap, "v") if v is None else v
    ro, rl, there = interpret.paged_attention(_np(q), k, v, n, m, present=present, **masks)
    scale = masks.get("scale") or q.shape[3] ** -0.5
    limit, lse_limit = _limits(_np(q), k, v, ro, max(n), c.dtype, scale)
    o, lse = _np(o), _np(lse)
    off = np.abs(o - ro)[there]
    assert (off <= limit[there]).all(), (off - limit[there]).max()
    # Half steps are spread evenly: 2 / sqrt(12) of the largest, norm-wise, at most.
    assert relative(o[there], ro[there]) <= 0.6 * HALF_STEP[c.dtype] + 2.0 ** -14
    empty = np.isneginf(rl) & there[..., None]
    assert (o[empty] == 0).all() and np.isneginf(lse[empty]).all()
    some = there[..., None] & ~empty
    assert (np.abs(lse[some] - rl[some]) <= lse_limit[some] + 2.0 ** -22 * np.abs(rl[some])).all()
    assert (o[~there] == was).all() and (lse[~there] == was).all()


CASES = [  # B, S, H, KV, D, page, cap, dtype, e4m3, outer, lengths, counts, masks
    (1, 1, 1, 1, 64, 1, 1, "bf16", False, False, [1], None, {}),
    (2, 1, 8, 2, 128, 16, 100, "bf16", False, False, [100, 31], None, {}),
    (3, 1, 4, 4, 64, 16, 64, "f16", False, True, [64, 32, 33], None, {}),
    (3, 1, 8, 2, 128, 16, 600, "bf16", True, False, [600, 1, 0], None, {}),
    (3, 1, 8, 2, 128, 24, 600, "f16", True, True, [127, 600, 129], None, {}),
    (2, 1, 16, 1, 256, 32, 300, "bf16", False, False, [300, 257], None, {}),
    (2, 1, 8, 1, 256, 5, 300, "f16", False, False, [300, 7], None, {}),
    (2, 1, 8, 1, 256, 64, 300, "bf16", True, False, [300, 200], None, {}),
    (2, 1, 6, 2, 8, 3, 50, "bf16", False, False, [50, 10], None, {}),
    (2, 1, 6, 2, 80, 7, 400, "bf16", False, False, [400, 222], None, {}),
    (2, 2, 6, 2, 96, 7, 400, "f16", True, False, [400, 222], None, {}),
    (2, 1, 6, 2, 192, 16, 200, "f16", False, False, [200, 77], None, {}),
    (2, 3, 4, 2, 224, 16, 200, "bf16", True, False, [200, 2], None, {}),
    (2, 4, 8, 2, 128, 16, 200, "bf16", False, False, [200, 3], None, {}),
    (3, 5, 6, 2, 64, 9, 300, "bf16", True, False, [300, 200, 5], [5, 2, 0], {}),
    (2, 5, 6, 2, 64, 9, 300, "bf16", False, False, [300, 4], None, {"causal": False}),
    (2, 4, 8, 2, 64, 7, 500, "f16", False, False, [500, 140], [4, 1], {"window": 100}),
    (2, 40, 4, 2, 64, 16, 300, "bf16", False, False, [300, 45], [40, 33], {}),
    (1, 40, 4, 1, 128, 16, 300, "bf16", True, False, [300], None, {"window": 17}),
    (1, 3, 32, 1, 64, 128, 1000, "f16", False, False, [1000], None, {}),
    (2, 1, 2, 2, 64, 16, 300, "bf16", False, False, [4000, -5], None, {}),
    (2, 1, 4, 2, 64, 16, 9000, "bf16", False, False, [9000, 1500], None, {"window": 1}),
    (40, 1, 8, 2, 128, 16, 700, "bf16", False, False, [(37 * i) % 701 for i in range(40)], None, {}),
    (1, 1, 8, 8, 64, 64, 9000, "bf16", True, False, [8999], None, {"scale": 0.3}),
    # Long tables: the keys divided among workgroups, pieces joined.
    (150, 1, 4, 1, 64, 64, 1600, "bf16", False, False, [(211 * i) % 1601 if i % 3 else 0 for i in range(150)], None, {}),
    (150, 1, 4, 1, 64, 64, 2600, "bf16", False, False, [(211 * i) % 2601 if i % 3 else 0 for i in range(150)], None, {}),
    (70, 2, 2, 1, 64, 7, 1500, "f16", True, False, [(97 * i) % 1501 for i in range(70)], [i % 3 for i in range(70)], {}),
    (3, 1, 16, 2, 256, 16, 1200, "f16", False, True, [1200, 0, 33], None, {}),
    (2, 3, 6, 2, 256, 32, 1000, "bf16", True, False, [1000, 999], [3, 2], {}),
    (2, 1, 4, 2, 224, 16, 1000, "bf16", True, True, [1000, 515], None, {}),
    (2, 4, 4, 2, 80, 5, 2500, "f16", False, False, [2500, 1], [4, 3], {"window": 1900}),
    (1, 1, 40, 2, 128, 128, 2000, "bf16", False, False, [1999], None, {}),
    (2, 20, 4, 1, 128, 16, 1500, "bf16", False, False, [1500, 37], [20, 11], {}),
    (2, 3, 4, 2, 128, 24, 1500, "bf16", True, False, [1411, 1500], None, {"causal": False}),
    (1, 1, 2, 1, 64, 1, 5000, "bf16", False, False, [4997], None, {}),
    (1, 2, 8, 2, 128, 1, 2900, "f16", True, True, [2900], None, {}),
    (1, 1, 1, 1, 128, 16, 40000, "bf16", True, False, [40000], None, {})]


@pytest.mark.parametrize("B,S,H,KV,D,page,cap,dtype,e4m3,outer,lengths,counts,masks", CASES)
def test_paged(target, B, S, H, KV, D, page, cap, dtype, e4m3, outer, lengths, counts, masks):
    announce("paged", B, S, H, KV, D, page, cap, dtype, e4m3, outer, lengths, counts, masks)
    c = Paged(B, cap, KV, D, page, dtype, e4m3, outer)
    gen = torch.Generator(device="cuda").manual_seed(D + cap)
    _fill(c, gen, cap)
    q = rows(gen, dtype, B, S, H, D, spread=False)
    o, lse = torch.full_like(q, 6.0), torch.full((B, S, H), 6.0, device="cuda")
    n, m = ints(*lengths), ints(*counts) if counts else None
    f = _attend(c, q, o, lse, n, m, **masks)
    f()
    torch.cuda.synchronize()
    _check(c, q, o, lse, n, m, was=6.0, **masks)
    o2 = torch.full_like(o, 6.0)
    _attend(c, q, o2, None, n, m, **masks)()  # without lse, the same bits
    torch.cuda.synchronize()
    assert torch.equal(o, o2)


@pytest.mark.parametrize("page,cap", [(16, 200), (7, 200), (16, 2000), (7, 2000)])
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 1])
def test_the_widest_windows(target, page, cap, window):
    """More new positions than a sequence holds, some of them below position 0: no
    window reaches past 32 bits there."""
    announce("paged widest window", page, cap, window)
    B, S, H, KV, D = 4, 9, 4, 2, 64
    c = Paged(B, cap, KV, D, page, "bf16", False)
    gen = torch.Generator(device="cuda").manual_seed(cap)
    _fill(c, gen, cap)
    q = rows(gen, "bf16", B, S, H, D, spread=False)
    n, m = ints(0, 3, cap, 1), ints(9, 7, 9, 5)
    o, lse = torch.full_like(q, 6.0), torch.full((B, S, H), 6.0, device="cuda")
    _attend(c, q, o, lse, n, m, window=window)()
    torch.cuda.synchronize()
    _check(c, q, o, lse, n, m, was=6.0, window=window)


@pytest.mark.parametrize("S,KV,cap", [(1, 700, 3600), (3, 300, 3600), (1, 4100, 3600)])
def test_more_sweeps_than_workgroups_at_once(target, S, KV, cap):
    """The keys in few pieces, down to one, that holds every sweep whole."""
    announce("paged many heads", S, KV, cap)
    B, D, page = 3, 8, 16
    c = Paged(B, cap, KV, D, page, "bf16", False)
    gen = torch.Generator(device="cuda").manual_seed(KV)
    _fill(c, gen, cap)
    q = rows(gen, "bf16", B, S, KV, D, spread=False)
    lengths = [cap, 0, 2077]
    n = ints(*lengths)
    o, lse = torch.full_like(q, 6.0), torch.full((B, S, KV), 6.0, device="cuda")
    _attend(c, q, o, lse, n)()
    torch.cuda.synchronize()
    assert (o[1] == 0).all() and torch.isneginf(lse[1]).all()
    for b in (0, 2):
        k, v = (t[c.table[b].long()].reshape(-1, KV, D)[:lengths[b]].double() for t in (c.k, c.v))
        for j in range(S):
            seen = lengths[b] - S + j + 1
            s = (k[:seen] * q[b, j].double()).sum(-1) * D ** -0.5
            w = torch.softmax(s, 0)
            want = torch.stack([(w * v[:seen, :, d]).sum(0) for d in range(D)], -1)
            score = (q[b, j].double().abs() * k.abs().amax(0)).sum(-1) * D ** -0.5 * ((D + 8) * 2.0 ** -24 + 2.0 ** -22)
            rel = 2 * (score + 2.0 ** -21 + (seen / 128 + 40) * 2.0 ** -24)
            limit = rel[:, None] * v.abs().amax(0) + 2.0 ** -8 * want.abs() + 2.0 ** -25
            assert ((o[b, j].double() - want).abs() <= limit).all()
            exact = torch.logsumexp(s, 0)
            assert ((lse[b, j].double() - exact).abs() <= score + 2.0 ** -20 + 2.0 ** -22 * exact.abs()).all()


@pytest.mark.parametrize("S,page,cap,e4m3", [(1, 16, 200, False), (5, 7, 200, True), (1, 7, 6000, True), (9, 16, 3000, False)])
def test_over_its_queries(target, S, page, cap, e4m3):
    announce("paged in place", S, page, cap, e4m3)
    B, H, KV, D = 3, 8, 2, 128
    c = Paged(B, cap, KV, D, page, "bf16", e4m3)
    gen = torch.Generator(device="cuda").manual_seed(cap)
    _fill(c, gen, cap)
    q = rows(gen, "bf16", B, S, H, D, spread=False)
    n, m = ints(cap, 0, cap // 2), ints(S, S, S - 1)
    o, lse = q.clone(), torch.empty((B, S, H), device="cuda")
    _attend(c, q, o, lse, n, m)()
    _attend(c, q, q, lse, n, m)()
    torch.cuda.synchronize()
    assert torch.equal(o, q)


@pytest.mark.parametrize("dtype,e4m3", [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("S,window,page,cap", [(1, 0, 8, 200), (4, 0, 8, 200), (4, 40, 8, 200), (9, 3, 8, 200), (1, 0, 16, 1600),
                                               (3, 0, 16, 1600), (3, 1500, 8, 1600), (4, 0, 16, 200)])
def test_what_no_query_sees_may_be_anything(target, dtype, e4m3, S, window, page, cap):
    """NaN and infinities behind the lengths, before the window, in the new
    rows of later positions and in pages no entry names (for the query that does not see them)."""
    announce("paged unseen", dtype, e4m3, S, window, page, cap)
    B, H, KV, D = 2, 4, 2, 64
    c = Paged(B, cap, KV, D, page, dtype, e4m3)
    gen = torch.Generator(device="cuda").manual_seed(S + window)
    _fill(c, gen, cap)
    q = rows(gen, dtype, B, S, H, D, spread=False)
    lengths = [150, 97] if cap == 200 else [1550, 1497]
    n = ints(*lengths)

    def run():
        o, lse = torch.full_like(q, 6.0), torch.full((B, S, H), 6.0, device="cuda")
        _attend(c, q, o, lse, n, window=window)()
        torch.cuda.synchronize()
        return o, lse
    o, lse = run()
    _check(c, q, o, lse, n, was=6.0, window=window)
    bad = 0x7f if e4m3 else float("nan")
    for b in range(B):
        for at in range(lengths[b], cap):  # behind the length
            for t in (c.k, c.v):
                t[c.where(b, at)] = bad
        if window:  # before every window
            for at in range(lengths[b] - S - window + 1):
                for t in (c.k, c.v):
                    t[c.where(b, at)] = bad
    used = set(c.table.cpu().view(-1).tolist())
    for page_ in set(range(c.pages)) - used:
        c.k[page_], c.v[page_] = bad, bad
    o2, lse2 = run()
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    # Each new row in turn, and the first key of the first window: only queries that see it know.
    for at in sorted({lengths[0] - 1 - i for i in range(S)} | {max(0, lengths[0] - S - window + 1 if window else 0)}):
        where = c.where(0, at)
        keep = c.k[where].clone(), c.v[where].clone()
        c.v[where] = bad
        if not e4m3:
            c.v[where][:, 1::2] = float("inf")
        o2, lse2 = run()
        assert torch.equal(o[1], o2[1]) and torch.equal(lse, lse2)
        for j in range(S):
            p = lengths[0] - S + j
            sees = at <= p and (not window or at > p - window)
            assert torch.equal(o[0, j], o2[0, j]) if not sees else not o2[0, j].isfinite().any(), (at, j)
        c.v[where] = keep[1]
        c.k[where] = bad
        o2, lse2 = run()
        for j in range(S):
            p = lengths[0] - S + j
            sees = at <= p and (not window or at > p - window)
            assert torch.equal(o[0, j], o2[0, j]) if not sees else o2[0, j].isnan().all(), (at, j)
        c.k[where] = keep[0]


@pytest.mark.parametrize("dtype,e4m3,page,cap,S", [("bf16", False, 8, 200, 2), ("f16", True, 8, 200, 2), ("bf16", True, 16, 2000, 1),
                                                    ("bf16", False, 16, 304, 1), ("f16", False, 7, 2100, 3)])
def test_entries_that_name_no_page(target, dtype, e4m3, page, cap, S):
    """No query sees a key there: holes in a sequence, one that has no page at all."""
    announce("paged bad pages", dtype, e4m3, page, cap, S)
    B, H, KV, D = 3, 4, 2, 64
    c = Paged(B, cap, KV, D, page, dtype, e4m3)
    gen = torch.Generator(device="cuda").manual_seed(3)
    _fill(c, gen, cap)
    c.table[0, 2], c.table[0, 3], c.table[0, 18], c.table[1] = -1, c.pages, 0x7fffffff, -0x80000000
    q = rows(gen, dtype, B, S, H, D, spread=False)
    o, lse = torch.full_like(q, 6.0), torch.full((B, S, H), 6.0, device="cuda")
    n = ints(150, 97, 200)
    table = c.table.cpu().numpy()
    present = (np.repeat(table, page, 1) >= 0) & (np.repeat(table, page, 1) < c.pages)
    _attend(c, q, o, lse, n)()
    torch.cuda.synchronize()
    _check(c, q, o, lse, n, present=present)
    assert (o[1] == 0).all() and torch.isneginf(lse[1]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_an_infinite_value_stays_one(target, dtype):
    announce("paged infinite", dtype)
    c = Paged(1, 500, 2, 64, 16, dtype)
    gen = torch.Generator(device="cuda").manual_seed(8)
    _fill(c, gen, 500)
    q = rows(gen, dtype, 1, 2, 4, 64, spread=False)
    q[0, 1] = 0.0  # every weight alike
    o, lse = torch.empty_like(q), torch.empty(1, 2, 4, device="cuda")
    n = ints(500)
    _attend(c, q, o, lse, n)()
    at, end = c.where(0, 3), c.where(0, 498)
    c.v[at][0, 5], c.v[end][1, 63] = float("inf"), -float("inf")
    o2, lse2 = torch.empty_like(o), torch.empty_like(lse)
    _attend(c, q, o2, lse2, n)()
    torch.cuda.synchronize()
    assert torch.isposinf(o2[0, :, :2, 5]).all() and torch.isneginf(o2[0, :, 2:, 63]).all()
    o2[0, :, :2, 5], o2[0, :, 2:, 63] = o[0, :, :2, 5], o[0, :, 2:, 63]
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype,e4m3", [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)])
def test_weights_hold_fp32s_bits(target, dtype, e4m3):
    """Keys in pairs, the second a step from the first in one feature, values v and -v: the output
    is the difference of weights about 2^-13 apart (fp16 2^-16, e4m3 2^-9).  fp32's score, exponential
    and sums leave each weight within about 2^-22, so 2^-9 (2^-6) of that difference; the
    result's rounding adds at most 2^-8.  Weights of 8 bits would leave it whole."""
    announce("paged weights", dtype, e4m3)
    B, H, KV, D, page, cap = 2, 8, 2, 128, 16, 1000
    c = Paged(B, cap, KV, D, page, dtype, e4m3)
    gen = torch.Generator(device="cuda").manual_seed(11)
    _fill(c, gen, cap)
    c.k[:, 1::2] = c.k[:, ::2]
    c.v[:, 1::2] = c.v[:, ::2] ^ 0x80 if e4m3 else -c.v[:, ::2]
    if e4m3:
        c.ks[:, 1::2], c.vs[:, 1::2] = c.ks[:, ::2], c.vs[:, ::2]
        x = c.k[:, 1::2, :, 0]
        c.k[:, 1::2, :, 0] = torch.where(x & 127 >= 126, x, x ^ 1)  # (126's neighbour is NaN)
    else:
        c.k[:, 1::2, :, 0] *= 1 + 2.0 ** (-7 if dtype == "bf16" else -10)
    q = rows(gen, dtype, B, 1, H, D, spread=False) * 0.25
    o, lse = torch.empty_like(q), torch.empty(B, 1, H, device="cuda")
    n = ints(1000, 500)
    _attend(c, q, o, lse, n)()
    torch.cuda.synchronize()
    ro, _, _ = interpret.paged_attention(_np(q), c.sequences(1008), c.sequences(1008, "v"), [1000, 500])
    assert relative(_np(o), ro) < (2.0 ** -5 if dtype == "f16" and not e4m3 else 2.0 ** -7), relative(_np(o), ro)


@pytest.mark.parametrize("f16", [False, True])
def test_every_code_is_the_value_it_stands_for(target, f16):
    """One key, so its weight is 1: every code at scales across fp16's (or bf16's) range comes out itself."""
    announce("paged codes", f16)
    dtype = "f16" if f16 else "bf16"
    grid = interpret.e4m3_values()
    codes = np.where(np.isnan(grid), 0, np.arange(256)).astype(np.uint8).reshape(1, 256)
    exponents = list(range(-14, 8)) if f16 else list(range(-117, 120, 4))
    B = len(exponents)
    c = Paged(B, 1, 1, 256, 1, dtype, True)
    for b, e in enumerate(exponents):
        at = c.where(b, 0)
        c.k[at], c.ks[at] = 0, 127
        c.v[at], c.vs[at] = torch.from_numpy(codes).cuda(), e + 127
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = rows(gen, dtype, B, 1, 1, 256, spread=False)
    o, lse = torch.empty_like(q), torch.empty(B, 1, 1, device="cuda")
    n = ints(*[1] * B)
    _attend(c, q, o, lse, n)()
    torch.cuda.synchronize()
    want = torch.from_numpy(c.sequences(1, "v")).to(TYPES[dtype])
    assert torch.equal(o.cpu(), want) and (lse == 0).all()


def test_strides_and_odd_addresses(target):
    """q and o in (B, H, S, D + 8) memory from an odd element; K and V side by side in one array."""
    import tempest_hip.launch as L
    announce("paged strides")
    B, S, H, KV, D, page, cap = 2, 3, 4, 2, 64, 8, 100
    c = Paged(B, cap, KV, D, page, "bf16")
    gen = torch.Generator(device="cuda").manual_seed(21)
    _fill(c, gen, cap)
    both = torch.stack([c.k, c.v], 3).contiguous()  # (pages, page, KV, 2, D)
    s = both.stride()
    cache = L.Cache(both.data_ptr(), both.data_ptr() + 2 * D, KV, D, page, c.pages, strides=(s[2], s[1], s[0]))
    q, o = (torch.zeros(B * H * S * (D + 8) + 1, device="cuda", dtype=torch.bfloat16)[1:].view(B, H, S, D + 8) for _ in range(2))
    q.copy_(torch.randn(q.shape, device="cuda", generator=gen))
    lse = torch.zeros(B, S, H, device="cuda")
    n = ints(100, 33)
    L.attention_paged(cache, B, H, S, q.data_ptr(), o.data_ptr(), c.table.data_ptr(), n.data_ptr(), c.width,
                      lse=lse.data_ptr(), q_strides=(q.stride(1), q.stride(2), q.stride(0)))()
    torch.cuda.synchronize()
    _check(c, q[..., :D].transpose(1, 2), o[..., :D].transpose(1, 2), lse, n)
    assert (o[..., D:] == 0).all()


def test_recorded_and_shared_workspaces(target):
    """Two recorded launches over one given workspace, replayed in turn with
    the lengths the device then holds, beside eager runs; every result its own eager one."""
    announce("paged graphs")
    cases = []
    for i, (D, e4m3, cap) in enumerate([(64, False, 3000), (128, True, 5000), (256, False, 3000)]):
        c = Paged(2, cap, 2, D, 16, "bf16", e4m3)
        gen = torch.Generator(device="cuda").manual_seed(i)
        _fill(c, gen, cap)
        q = rows(gen, "bf16", 2, 1, 8, D, spread=False)
        o, lse, n = torch.empty_like(q), torch.empty(2, 1, 8, device="cuda"), ints(cap, cap // 2)
        cases.append((c, q, o, lse, n, _attend(c, q, o, lse, n)))
    size = max(f.workspace() for *_, f in cases)
    assert size > 0
    space = torch.full((size,), 255, device="cuda", dtype=torch.uint8)
    for *_, f in cases:
        f.set_workspace(space.data_ptr())
    graphs = [target.capture([f] * 20) for *_, f in cases]
    for lengths in ([1, 2999], [0, 128], [3000, 129], [777, 2500]):
        for (c, q, o, lse, n, f), graph in zip(cases, graphs):
            n.copy_(torch.tensor(lengths, dtype=torch.int32))
            target.replay(graph)
        space.fill_(255)  # nothing of one run is kept for the next
        for (c, q, o, lse, n, f), graph in zip(cases, graphs):
            target.replay(graph)
            torch.cuda.synchronize()
            got = o.clone(), lse.clone()
            _check(c, q, o, lse, n)
            o.fill_(3.0)
            f()
            torch.cuda.synchronize()
            assert torch.equal(o, got[0]) and torch.equal(lse, got[1])


def test_a_cache_past_32_bits(target):
    """A page whose elements lie past 2^32 of the arrays' start."""
    import tempest_hip.launch as L
    announce("paged past 2^32")
    KV, D, page, pages = 8, 256, 64, 33000
    k = torch.zeros(pages, page, KV, D, device="cuda", dtype=torch.bfloat16)  # 4.3e9 elements, 8.7 GB
    c = Paged(1, 130, KV, D, page, "bf16", spare=0)
    gen = torch.Generator(device="cuda").manual_seed(2)
    _fill(c, gen, 130)
    table = ints(32999, 32950, 5)
    both = k, k.clone()
    for i, at in enumerate([32999, 32950, 5]):
        both[0][at], both[1][at] = c.k[int(c.table[0, i])], c.v[int(c.table[0, i])]
    q = rows(gen, "bf16", 1, 1, 8, D, spread=False)
    o, lse, n = torch.empty_like(q), torch.empty(1, 1, 8, device="cuda"), ints(130)
    cache = L.Cache(both[0].data_ptr(), both[1].data_ptr(), KV, D, page, pages)
    L.attention_paged(cache, 1, 8, 1, q.data_ptr(), o.data_ptr(), table.data_ptr(), n.data_ptr(), 3, lse=lse.data_ptr())()
    torch.cuda.synchronize()
    _check(c, q, o, lse, n)


@pytest.mark.parametrize("dtype,e4m3,page", [("bf16", False, 16), ("bf16", True, 7), ("f16", True, 32)])
def test_decoding_as_it_is_used(target, dtype, e4m3, page):
    """A prompt and then single tokens, each step turned by its positions,
    written and attended from one recording, lengths counted up on the device;
    the prompt's context read back and attended densely gives the same."""
    import tempest_hip.launch as L
    announce("paged decoding", dtype, e4m3, page)
    B, H, KV, D, prompt, steps = 2, 8, 2, 64, 37, 6
    cap = prompt + steps
    c = Paged(B, cap, KV, D, page, dtype, e4m3)
    gen = torch.Generator(device="cuda").manual_seed(31)
    freqs = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().cuda()
    n = ints(0, 0)
    held = {"k": np.zeros((B, cap, KV, D)), "v": np.zeros((B, cap, KV, D))}

    def program(S):
        q, k, v = (rows(gen, dtype, B, S, h, D, spread=False) for h in (H, KV, KV))
        yq, yk, o, lse = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q), torch.empty(B, S, H, device="cuda")
        at = torch.zeros(B, S, 1, device="cuda", dtype=torch.int32)
        p = lambda *ts: [t.data_ptr() for t in ts]  # noqa: E731
        return (q, k, v, yq, yk, o, lse, at), [
            L.rotary(B, S, H, KV, D, *p(q, k, yq, yk, at, freqs), dtype=c.type),
            L.cache_write(c.cache, B, S, *p(yk, v, c.table, n), c.width, dtype=c.type),
            _attend(c, yq, o, lse, n)]

    def step(arrays, run, S):
        q, k, v, yq, yk, o, lse, at = arrays
        for t in (q, k, v):
            t.copy_(rows(gen, dtype, *t.shape, spread=False))
        start = int(n[0])
        at.copy_(torch.arange(start, start + S, device="cuda")[None, :, None].expand(B, S, 1))
        n.add_(S)
        run()
        torch.cuda.synchronize()
        for name, x in (("k", yk), ("v", v)):
            x = _np(x)
            held[name][:, start:start + S] = interpret.e4m3_held(*interpret.e4m3_rows(x, dtype == "f16")) if e4m3 else x
        want = interpret.rotary(_np(q), at.cpu().numpy(), freqs.cpu().numpy(), [D // 2])
        assert np.abs(_np(yq) - want).max() < 2.0 ** -7 * np.abs(want).max()
        _check(c, yq, o, lse, n, k=held["k"][:, :cap], v=held["v"][:, :cap])

    arrays, launches = program(prompt)
    step(arrays, lambda: [f() for f in launches], prompt)
    if dtype == "bf16":  # the dense forward over what is read back
        _, _, _, yq, _, o, lse, _ = arrays
        k, v = (torch.zeros(B, prompt, KV, D, device="cuda", dtype=TYPES[dtype]) for _ in range(2))
        L.cache_read(c.cache, B, prompt, k.data_ptr(), v.data_ptr(), c.table.data_ptr(), n.data_ptr(), c.width, dtype=c.type)()
        o2, lse2 = torch.empty_like(o), torch.empty_like(lse)
        L.attention_fwd(B, H, KV, prompt, yq.data_ptr(), k.data_ptr(), v.data_ptr(), o2.data_ptr(), lse2.data_ptr(),
                        causal=True, head_dim=D)()
        torch.cuda.synchronize()
        assert (o.float() - o2.float()).abs().max() < 2.0 ** -5 and (lse - lse2).abs().max() < 1e-4
    arrays, launches = program(1)
    graph = target.capture(launches)
    for _ in range(steps):
        step(arrays, lambda: target.replay(graph), 1)


@pytest.mark.parametrize("dtype,e4m3", [("f16", False), ("bf16", False), ("f16", True), ("bf16", True)])
@pytest.mark.parametrize("S,page,cap", [(1, 16, 200), (2, 7, 300), (1, 16, 2500), (3, 7, 2500)])
def test_small_weights_beside_a_large_one(target, dtype, e4m3, S, page, cap):
    """One key of score 32 whose value is 0, the others between -4 and 6 with values up to thousands: the
    output is the small weights' alone, 2^-37 to 2^-52 of the large one.  Each is within `score` +
    2^-21 of itself as everywhere (the scores' own products are exact), so the weighted mean within twice that
    of the weighted sizes of the values, 0 for the large one's."""
    announce("paged small weights", dtype, e4m3, S, page, cap)
    B, H, KV, D = 2, 4, 2, 64
    c = Paged(B, cap, KV, D, page, dtype, e4m3)
    gen = torch.Generator(device="cuda").manual_seed(cap + S)
    k, v = torch.zeros(c.pages, page, KV, D, device="cuda"), rows(gen, dtype, c.pages, page, KV, D, spread=False).float().abs() * 2.0 ** 12
    k[..., 0] = torch.rand(k.shape[:-1], device="cuda", generator=gen) * 10 - 4
    for b in range(B):
        k[c.where(b, 5)][:, 0], v[c.where(b, 5)] = 32.0, 0.0
    for name, x in (("k", k), ("v", v)):
        x = x.to(TYPES[dtype])
        if e4m3:
            codes, scales = interpret.e4m3_rows(_np(x), dtype == "f16")
            getattr(c, name).copy_(torch.from_numpy(codes))
            getattr(c, name + "s").copy_(torch.from_numpy(scales))
        else:
            getattr(c, name).copy_(x)
    q = torch.zeros(B, S, H, D, device="cuda", dtype=TYPES[dtype])
    q[..., 0] = 1.0
    o, lse = torch.empty_like(q), torch.empty(B, S, H, device="cuda")
    n = [cap, cap - 31]
    _attend(c, q, o, lse, ints(*n), scale=1.0)()
    torch.cuda.synchronize()
    k, v = c.sequences(cap), c.sequences(cap, "v")
    want, _, _ = interpret.paged_attention(_np(q), k, v, n, scale=1.0)
    size, _, _ = interpret.paged_attention(_np(q), k, np.abs(v), n, scale=1.0)
    score = 32.0 * ((D + 8) * 2.0 ** -24 + 2.0 ** -22)
    limit = 2 * (score + 2.0 ** -21 + (cap / 128 + 40) * 2.0 ** -24) * size + HALF_STEP[dtype] * np.abs(want)
    limit += 2.0 ** -25 if dtype == "f16" else 0.0  # (half a step below fp16's normals)
    off = np.abs(_np(o) - want)
    assert (want[..., 1:] > 0).all() and (off <= limit).all(), (off / limit).max()
    if not e4m3:  # infinite values under small weights: infinite outputs, the others' bits as they were
        o2, lse2 = torch.empty_like(o), torch.empty_like(lse)
        c.v[c.where(0, 7)][0, 9], c.v[c.where(1, cap - 60)][1, 40] = float("inf"), -float("inf")
        _attend(c, q, o2, lse2, ints(*n), scale=1.0)()
        torch.cuda.synchronize()
        assert torch.isposinf(o2[0, :, :2, 9]).all() and torch.isneginf(o2[1, :, 2:, 40]).all()
        o2[0, :, :2, 9], o2[1, :, 2:, 40] = o[0, :, :2, 9], o[1, :, 2:, 40]
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("page", [1, 16])
def test_every_fp16_value_comes_out_itself(target, page):
    """One key, so its weight is 1: every finite value, both infinities and every NaN."""
    announce("paged fp16 values", page)
    codes = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(256, 1, 1, 256).view(torch.float16)
    c = Paged(256, 1, 1, 256, page, "f16")
    c.k.zero_()
    for b in range(256):
        c.v[c.where(b, 0)] = codes[b, 0].cuda()
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = rows(gen, "f16", 256, 1, 1, 256, spread=False)
    o, n = torch.empty_like(q), ints(*[1] * 256)
    _attend(c, q, o, None, n)()
    torch.cuda.synchronize()
    o, want = o.cpu(), codes.view(256, 1, 1, 256)
    assert torch.equal(o.isnan(), want.isnan())
    assert torch.equal(o[~want.isnan()], want[~want.isnan()])


@pytest.mark.parametrize("cap", [200, 3000])
def test_repointed_to_odd_elements(target, cap):
    """q and o at an odd element, given after the launch was built; the cache's arrays stay at 16 bytes."""
    from tempest_hip import HIPError
    announce("paged odd elements", cap)
    B, S, H, KV, D = 2, 2, 4, 2, 64
    c = Paged(B, cap, KV, D, 16, "bf16")
    gen = torch.Generator(device="cuda").manual_seed(cap)
    _fill(c, gen, cap)
    q, o, lse = rows(gen, "bf16", B, S, H, D, spread=False), torch.zeros(B, S, H, D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, S, H, device="cuda")
    n = ints(cap, cap // 3)
    f = _attend(c, q, o, lse, n)
    q2 = rows(gen, "bf16", B, S, H, D, spread=False, offset=3)
    o2 = torch.zeros(B * S * H * D + 1, device="cuda", dtype=torch.bfloat16)[1:].view(B, S, H, D)
    f.repoint("q", q2.data_ptr())
    f.repoint("o", o2.data_ptr())
    f()
    torch.cuda.synchronize()
    _check(c, q2, o2, lse, n)
    for name, at in (("q", q2.data_ptr() + 1), ("table", c.table.data_ptr() + 2), ("v_cache", c.v.data_ptr() + 8)):
        with pytest.raises(HIPError):
            f.repoint(name, at)


@pytest.mark.parametrize("cap", [640, 720, 800])
def test_the_split_goes_by_positions_and_features(target, cap):
    """Whether a sweep is one workgroup's is the same for pages in sixteens and others, and for all head
    dims that one kernel takes."""
    announce("paged split", cap)
    ways = set()
    for page, D in ((16, 128), (8, 128), (5, 128), (16, 80), (10, 96)):
        c = Paged(1, cap, 8, D, page, "bf16")
        q = torch.zeros(1, 1, 32, D, device="cuda", dtype=torch.bfloat16)
        ways.add("whole" in _attend(c, q, torch.zeros_like(q), None, ints(cap)).describe())
    assert len(ways) == 1


@pytest.mark.parametrize("B,H,KV,D,page,cap,dtype,e4m3,window", [
    (100, 2, 1, 8, 1, 2300, "bf16", False, 0), (100, 2, 1, 64, 1, 2400, "f16", False, 2200), (100, 4, 1, 32, 1, 2700, "bf16", True, 0)])
def test_whole_sweeps_of_more_entries_than_lds_holds(target, B, H, KV, D, page, cap, dtype, e4m3, window):
    """2048 entries of the table are in LDS at a time: sweeps that take them in two parts, from wherever they start."""
    lengths = [(211 * i) % (cap + 1) if i % 3 else cap - i for i in range(B)]
    c = Paged(1, 1, KV, D, 1, dtype, e4m3)
    q = torch.zeros(B, 1, H, D, device="cuda", dtype=TYPES[dtype])
    import tempest_hip.launch as L
    assert "whole" in L.attention_paged(c.cache, B, H, 1, q.data_ptr(), q.data_ptr(), c.table.data_ptr(), c.table.data_ptr(), cap,
                                        window=window, dtype=c.type).describe()
    test_paged(target, B, 1, H, KV, D, page, cap, dtype, e4m3, False, lengths, None, {"window": window} if window else {})


@pytest.mark.parametrize("B,S,KV,D,page,cap,dtype,e4m3,window", [
    (3, 1, 1100, 8, 1, 3600, "bf16", False, 0), (3, 1, 1100, 8, 1, 3600, "f16", False, 3100), (4, 1, 1100, 8, 2, 5000, "bf16", False, 0),
    (3, 2, 1100, 8, 1, 3600, "bf16", False, 0), (3, 1, 1100, 32, 1, 3600, "bf16", True, 0), (2, 1, 2100, 64, 1, 2600, "bf16", False, 0)])
def test_pieces_of_more_entries_than_lds_holds(target, B, S, KV, D, page, cap, dtype, e4m3, window):
    """The same where the keys are cut in a few pieces of thousands of positions."""
    announce("paged long pieces", B, S, KV, D, page, cap, dtype, e4m3, window)
    c = Paged(B, cap, KV, D, page, dtype, e4m3)
    gen = torch.Generator(device="cuda").manual_seed(cap + D)
    if e4m3:  # any codes but NaN's, scales 2^-8..2^-6
        for t, s in ((c.k, c.ks), (c.v, c.vs)):
            t.copy_(torch.randint(0, 127, t.shape, device="cuda", generator=gen) + 128 * torch.randint(0, 2, t.shape, device="cuda", generator=gen))
            s.copy_(torch.randint(119, 122, s.shape, device="cuda", generator=gen))
    else:
        _fill(c, gen, cap)
    q = rows(gen, dtype, B, S, KV, D, spread=False)
    lengths = [cap - 500 * (b % 2) - b for b in range(B)]
    n = ints(*lengths)
    o, lse = torch.full_like(q, 6.0), torch.full((B, S, KV), 6.0, device="cuda")
    _attend(c, q, o, lse, n, window=window)()
    torch.cuda.synchronize()

    def held(t, s, b, heads):
        x = t[c.table[b].long()].reshape(-1, KV, t.shape[-1])[:lengths[b], heads]
        if not e4m3:
            return x.double()
        s = s[c.table[b].long()].reshape(-1, KV, s.shape[-1])[:lengths[b], heads].double()
        return (x.view(torch.float8_e4m3fn).double().unflatten(-1, (-1, 32)) * torch.exp2(s - 127)[..., None]).flatten(-2)
    for b in range(B):
        for h in range(0, KV, 300):
            heads = slice(h, min(KV, h + 300))
            k, v = held(c.k, c.ks, b, heads), held(c.v, c.vs, b, heads)
            for j in range(S):
                end = lengths[b] - S + j + 1
                lo = max(0, end - window) if window else 0
                qj = q[b, j, heads].double()
                s = (k[lo:end] * qj).sum(-1) * D ** -0.5
                w = torch.softmax(s, 0)
                want = (w[..., None] * v[lo:end]).sum(0)
                score = (qj.abs() * k.abs().amax(0)).sum(-1) * D ** -0.5 * ((D + 8) * 2.0 ** -24 + 2.0 ** -22)
                rel = 2 * (score + 2.0 ** -21 + (end / 128 + 40) * 2.0 ** -24)
                limit = rel[:, None] * v.abs().amax(0) + HALF_STEP[dtype] * want.abs() + 2.0 ** -25
                assert ((o[b, j, heads].double() - want).abs() <= limit).all(), (b, h, j)
                exact = torch.logsumexp(s, 0)
                assert ((lse[b, j, heads].double() - exact).abs() <= score + 2.0 ** -20 + 2.0 ** -22 * exact.abs()).all(), (b, h, j)


@pytest.mark.parametrize("B,S,H,KV,D,page,cap,dtype,e4m3,lengths,counts,masks", [
    (2, 1000, 4, 2, 64, 16, 1500, "bf16", False, [1500, 900], [1000, 777], {}),
    (1, 2500, 2, 1, 128, 16, 3100, "bf16", True, [3100], [2499], {"window": 700}),
    (2, 700, 6, 2, 64, 7, 1500, "f16", False, [1499, 20], [700, 33], {}),
    (2, 300, 4, 1, 256, 24, 700, "bf16", False, [700, 300], None, {"causal": False}),
    (2, 65535, 1, 1, 8, 16, 400, "bf16", False, [300, 400], [300, 0], {}),
    (1, 65535, 3, 1, 96, 16, 400, "f16", True, [390], [37], {"window": 50})])
def test_many_new_positions(target, B, S, H, KV, D, page, cap, dtype, e4m3, lengths, counts, masks):
    """A prompt's next piece over its context: many tiles of rows a head, ragged counts, the most positions there may be."""
    test_paged(target, B, S, H, KV, D, page, cap, dtype, e4m3, False, lengths, counts, masks)
