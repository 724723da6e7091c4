"""Rotary positions through th_build_rotary against the float64 oracle, every
element: the angle is formed in fp64 (off by 2^-51 of its turns at most), sin and
cos are within 2^-23 (fp32's last place twice), the two products and their sum add three roundings of
2^-24, so with |u|, |v| the pair's values an element is off by at most
2^-21.5 (|u| + |v|), and by half a step of its type."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import interpret

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _np(t):
    return t.double().cpu().numpy()


def _dtype(name):
    import tempest_hip.launch as L
    return {"f32": L.F32, "bf16": L.BF16, "f16": L.F16}[name]


def _array(gen, dt, *shape, offset=0):
    n = int(np.prod(shape))
    t = torch.empty(n + offset, device="cuda", dtype=dt)[offset:].view(*shape)
    return t.copy_(torch.randn(*shape, device="cuda", generator=gen))


def _freqs(n):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)).float().cuda()


def _check(got, x, positions, freqs, sections, pairs, inverse, dtype):
    x64, want = _np(x), interpret.rotary(_np(x), positions.cpu().numpy(), freqs.cpu().numpy(), sections, pairs, inverse)
    n = len(freqs)
    size = np.abs(x64)
    if pairs:
        size[..., :2 * n] = np.repeat(size[..., 0:2 * n:2] + size[..., 1:2 * n:2], 2, -1)
    else:
        size[..., :2 * n] = np.tile(size[..., :n] + size[..., n:2 * n], 2)
    off = np.abs(_np(got) - want)
    limit = 2.0 ** -21.5 * size + HALF_STEP[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 0)
    assert (off <= limit).all(), (off - limit).max()
    assert np.array_equal(_np(got)[..., 2 * n:], x64[..., 2 * n:])


@pytest.mark.parametrize("B,S,H,KV,D,R,sections,pairs,inverse,dtype,offset", [
    (1, 1, 1, 0, 2, 2, [1], False, False, "f32", 0),
    (16, 1, 32, 8, 128, 128, [64], False, False, "bf16", 0),
    (2, 37, 5, 1, 128, 128, [16, 24, 24], False, False, "bf16", 0),
    (2, 37, 4, 2, 128, 128, [16, 24, 24], True, True, "f16", 0),
    (3, 129, 3, 3, 64, 32, [7, 9], True, False, "bf16", 3),
    (1, 100, 2, 2, 80, 80, [20, 20], False, True, "f32", 1),
    (2, 11, 6, 2, 96, 24, [0, 5, 7, 0], False, False, "f16", 1),
    (1, 300, 1, 1, 7, 6, [3], True, False, "bf16", 0),
    (1, 9, 2, 1, 1024, 1024, [512], False, False, "f32", 0),
    (1, 3, 300, 0, 256, 64, [32], False, True, "bf16", 0),
    (2, 4096, 8, 2, 64, 64, [32], True, False, "bf16", 0)])
def test_rotary(target, B, S, H, KV, D, R, sections, pairs, inverse, dtype, offset):
    import tempest_hip.launch as L
    announce("rotary", B, S, H, KV, D, R, sections, pairs, inverse, dtype, offset)
    gen = torch.Generator(device="cuda").manual_seed(S + D)
    dt = TYPES[dtype]
    q, k = _array(gen, dt, B, S, H, D, offset=offset), _array(gen, dt, B, S, max(KV, 1), D, offset=offset)
    positions = torch.randint(0, 1 << 20, (B, S, len(sections)), dtype=torch.int32, device="cuda", generator=gen)
    freqs = _freqs(R // 2)
    yq, yk = (torch.full_like(x, 7.0) for x in (q, k))
    f = L.rotary(B, S, H, KV, D, q.data_ptr(), k.data_ptr(), yq.data_ptr(), yk.data_ptr(), positions.data_ptr(),
                 freqs.data_ptr(), sections=sections, rotary_dim=R, pairs=pairs, inverse=inverse, dtype=_dtype(dtype))
    keep = q.clone(), k.clone()
    f()
    torch.cuda.synchronize()
    _check(yq, q, positions, freqs, sections, pairs, inverse, dtype)
    if KV:
        _check(yk, k, positions, freqs, sections, pairs, inverse, dtype)
    else:
        assert (yk == 7.0).all()
    assert torch.equal(q, keep[0]) and torch.equal(k, keep[1])
    # In place the same bits.
    L.rotary(B, S, H, KV, D, q.data_ptr(), k.data_ptr(), q.data_ptr(), k.data_ptr(), positions.data_ptr(),
             freqs.data_ptr(), sections=sections, rotary_dim=R, pairs=pairs, inverse=inverse, dtype=_dtype(dtype))()
    torch.cuda.synchronize()
    assert torch.equal(q, yq) and (not KV or torch.equal(k, yk))


def test_rotary_strides_and_broadcast_positions(target):
    """q and k as parts of one array of all heads, written to arrays of other
    orders; one row of positions for the whole batch, its axes apart; the
    elements between rows stay."""
    import tempest_hip.launch as L
    announce("rotary strides")
    B, S, H, KV, D, R = 3, 21, 4, 2, 64, 48
    gen = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(B, S, H + 2 * KV, D, device="cuda", generator=gen).to(torch.bfloat16)
    q, k = qkv[:, :, :H], qkv[:, :, H:H + KV]
    yq = torch.full((B, H, S, D + 8), 3.0, device="cuda", dtype=torch.bfloat16)
    yk = torch.full((S, B, KV, D), 3.0, device="cuda", dtype=torch.bfloat16)
    positions = torch.randint(-50, 5000, (2, S), dtype=torch.int32, device="cuda", generator=gen)
    freqs = _freqs(R // 2)
    st = lambda t, order: [t.stride(i) for i in order]  # noqa: E731
    L.rotary(B, S, H, KV, D, q.data_ptr(), k.data_ptr(), yq.data_ptr(), yk.data_ptr(), positions.data_ptr(),
             freqs.data_ptr(), sections=[10, 14], rotary_dim=R, q_strides=st(q, (2, 1, 0)), k_strides=st(k, (2, 1, 0)),
             q_out_strides=st(yq, (1, 2, 0)), k_out_strides=st(yk, (2, 0, 1)), position_strides=(S, 1, 0))()
    torch.cuda.synchronize()
    full = positions.t()[None].expand(B, S, 2)
    _check(yq[..., :D].transpose(1, 2), q, full, freqs, [10, 14], False, False, "bf16")
    _check(yk.transpose(0, 1), k, full, freqs, [10, 14], False, False, "bf16")
    assert (yq[..., D:] == 3.0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rotary_repointed_to_odd_elements(target, dtype):
    import tempest_hip.launch as L
    from tempest_hip import HIPError
    announce("rotary odd elements", dtype)
    B, S, H, KV, D = 2, 9, 4, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(6)
    dt = TYPES[dtype]
    q, k, yq, yk = (_array(gen, dt, B, S, n, D) for n in (H, KV, H, KV))
    positions = torch.randint(0, 9000, (B, S, 1), dtype=torch.int32, device="cuda", generator=gen)
    freqs = _freqs(32)
    f = L.rotary(B, S, H, KV, D, q.data_ptr(), k.data_ptr(), yq.data_ptr(), yk.data_ptr(), positions.data_ptr(),
                 freqs.data_ptr(), dtype=_dtype(dtype))
    odd = {n: _array(gen, dt, B, S, h, D, offset=at) for n, h, at in (("q", H, 1), ("k", KV, 3), ("q_out", H, 5), ("k_out", KV, 1))}
    for n, t in odd.items():
        f.repoint(n, t.data_ptr())
    f()
    torch.cuda.synchronize()
    _check(odd["q_out"], odd["q"], positions, freqs, [32], False, False, dtype)
    _check(odd["k_out"], odd["k"], positions, freqs, [32], False, False, dtype)
    for n in ("q", "positions", "freqs"):  # between elements there is none
        with pytest.raises(HIPError):
            f.repoint(n, q.data_ptr() + (1 if n == "q" else 2))


def test_rotary_far_positions(target):
    """Positions across all of int32 keep their turn: at 2^31 of the first
    pair 3.4e8 turns, fp64 leaves 2^-24 of one (the oracle's own angle, in radians, as much)."""
    import tempest_hip.launch as L
    announce("rotary far")
    at = torch.tensor([0, 1, -1, 1 << 24, (1 << 24) + 1, 1 << 30, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32, device="cuda")
    x = torch.zeros(1, len(at), 1, 64, device="cuda")
    x[..., :32] = 1.0
    freqs = _freqs(32)
    y = torch.empty_like(x)
    L.rotary(1, len(at), 1, 0, 64, x.data_ptr(), 0, y.data_ptr(), 0, at.data_ptr(), freqs.data_ptr(), dtype=L.F32)()
    torch.cuda.synchronize()
    want = interpret.rotary(_np(x), at.cpu().numpy()[None, :, None], freqs.cpu().numpy(), [32])
    assert np.abs(_np(y) - want).max() < 2.0 ** -21  # 2^-23 a cosine, 2 * 2 pi 2^-53 2^28.4 its angle
    assert torch.equal(y[0, 0], x[0, 0])


def test_rotary_gradient_of_a_graph(target):
    """Forward and gradient captured and replayed over moved arrays and new
    positions: sum(rotary(x) .* g) has the gradient the inverse turn gives, and
    turning back what was turned gives x again."""
    import tempest_hip.launch as L
    announce("rotary graph")
    B, S, H, KV, D = 2, 65, 4, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(9)
    new = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    q, k, yq, yk, zq, zk = (new(B, S, n, D) for n in (H, KV, H, KV, H, KV))
    positions = torch.randint(0, 9000, (B, S, 1), dtype=torch.int32, device="cuda", generator=gen)
    freqs = _freqs(32)
    p = lambda *ts: [t.data_ptr() for t in ts]  # noqa: E731
    fwd = L.rotary(B, S, H, KV, D, *p(q, k, yq, yk, positions, freqs), dtype=L.F32)
    back = L.rotary(B, S, H, KV, D, *p(yq, yk, zq, zk, positions, freqs), inverse=True, dtype=L.F32)
    graph = target.capture([fwd, back])
    for i in range(3):
        q.copy_(new(B, S, H, D))
        positions.copy_(torch.randint(0, 1 << 18, positions.shape, dtype=torch.int32, device="cuda", generator=gen))
        target.replay(graph)
        torch.cuda.synchronize()
        _check(yq, q, positions, freqs, [32], False, False, "f32")
        _check(zk, yk, positions, freqs, [32], False, True, "f32")
        assert (zq - q).abs().max() < 2.0 ** -20 * 8  # two turns of values under 6
    q2 = new(B, S, H, D)
    fwd.repoint("q", q2.data_ptr())
    fwd()
    torch.cuda.synchronize()
    _check(yq, q2, positions, freqs, [32], False, False, "f32")


@pytest.mark.parametrize("dtype,D,R,H,KV,pairs", [("bf16", 64, 32, 4, 2, False), ("f32", 80, 20, 3, 0, True),
                                                  ("f16", 7, 6, 2, 1, True), ("bf16", 256, 64, 40, 8, False)])
def test_rotary_moves_between_in_place_and_apart(target, dtype, D, R, H, KV, pairs):
    """Built in place with part of a head turned, then pointed at another q_out and k_out, at another
    q and k, and back: the features that pass are in every result.  And built apart, then in place."""
    import tempest_hip.launch as L
    announce("rotary moves", dtype, D, R, H, KV, pairs)
    B, S = 2, 37
    gen = torch.Generator(device="cuda").manual_seed(D + R)
    dt = TYPES[dtype]
    x = {"q": _array(gen, dt, B, S, H, D), "k": _array(gen, dt, B, S, max(KV, 1), D)}
    positions = torch.randint(0, 1 << 16, (B, S, 1), dtype=torch.int32, device="cuda", generator=gen)
    freqs = _freqs(R // 2)

    def launch(a, y):
        return L.rotary(B, S, H, KV, D, a["q"].data_ptr(), a["k"].data_ptr(), y["q"].data_ptr(), y["k"].data_ptr(),
                        positions.data_ptr(), freqs.data_ptr(), rotary_dim=R, pairs=pairs, dtype=_dtype(dtype))

    def held(y):
        torch.cuda.synchronize()
        for n in ("q", "k") if KV else ("q",):
            _check(y[n], x[n], positions, freqs, [R // 2], pairs, False, dtype)

    def copies():
        return {n: t.clone() for n, t in x.items()}

    def empty():
        return {n: torch.full_like(t, 7.0) for n, t in x.items()}
    a = copies()
    f = launch(a, a)
    f()
    held(a)
    a, y = copies(), empty()
    for n in ("q", "k"):
        f.repoint(n, a[n].data_ptr())
        f.repoint(n + "_out", y[n].data_ptr())
    f()
    held(y)
    assert torch.equal(a["q"], x["q"]) and torch.equal(a["k"], x["k"])
    b = copies()  # q and k elsewhere, where one stays in place: both results whole
    f.repoint("q_out", a["q"].data_ptr())
    f.repoint("k", b["k"].data_ptr())
    y["k"].fill_(7.0)
    f()
    held({"q": a["q"], "k": y["k"]})
    a, y = copies(), empty()
    g = launch(a, y)
    for n in ("q", "k"):
        g.repoint(n + "_out", a[n].data_ptr())
    g()
    held(a)
    assert (y["q"] == 7.0).all() and (y["k"] == 7.0).all()
