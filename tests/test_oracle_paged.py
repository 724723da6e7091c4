"""The oracle's rotary positions, e4m3 rows and paged attention, pinned on the
CPU: turns against complex numbers and their invariants, codes against
torch's conversion and the definition, attention against torch float64."""
import numpy as np
import pytest
import torch

from oracle import interpret


def _rng(seed=0):
    return np.random.default_rng(seed)


@pytest.mark.parametrize("pairs", [False, True])
def test_rotary_is_a_turn_of_each_pair(pairs):
    r = _rng()
    x = r.standard_normal((2, 5, 3, 16))
    positions = r.integers(0, 1000, (2, 5, 2))
    freqs = 10000.0 ** (-np.arange(6) / 6)
    y = interpret.rotary(x, positions, freqs, [2, 4], pairs)
    z = x[..., :12].reshape(2, 5, 3, 6, 2) if pairs else np.stack([x[..., :6], x[..., 6:12]], -1)
    theta = np.concatenate([positions[..., :1] * freqs[:2], positions[..., 1:] * freqs[2:]], -1)[:, :, None]
    w = (z[..., 0] + 1j * z[..., 1]) * np.exp(1j * theta)
    got = y[..., :12].reshape(2, 5, 3, 6, 2) if pairs else np.stack([y[..., :6], y[..., 6:12]], -1)
    assert np.allclose(got[..., 0], w.real, atol=1e-13) and np.allclose(got[..., 1], w.imag, atol=1e-13)
    assert np.array_equal(y[..., 12:], x[..., 12:])
    back = interpret.rotary(y, positions, freqs, [2, 4], pairs, inverse=True)
    assert np.allclose(back, x, atol=1e-13)
    # The gradient of sum(y .* g): turned back, as differences say.
    g = r.standard_normal(x.shape)
    dx = interpret.rotary(g, positions, freqs, [2, 4], pairs, inverse=True)
    d = r.standard_normal(x.shape)
    f = lambda t: (interpret.rotary(x + t * d, positions, freqs, [2, 4], pairs) * g).sum()  # noqa: E731
    assert np.isclose((f(0.5) - f(-0.5)), (dx * d).sum(), rtol=1e-12)


def test_rotary_scores_depend_on_distance():
    r = _rng(1)
    q, k = r.standard_normal((1, 1, 1, 8)), r.standard_normal((1, 1, 1, 8))
    freqs = 10000.0 ** (-np.arange(4) / 4)
    turn = lambda x, p: interpret.rotary(x, np.full((1, 1, 1), p), freqs, [4])  # noqa: E731
    assert np.isclose((turn(q, 17) * turn(k, 5)).sum(), (turn(q, 1012) * turn(k, 1000)).sum(), rtol=1e-11)


def test_e4m3_values_are_torchs():
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(interpret.e4m3_values(), want, equal_nan=True)


def test_e4m3_rows():
    r = _rng(2)
    x = np.concatenate([r.standard_normal((40, 64)) * 2.0 ** r.integers(-30, 30, (40, 1)),
                        r.integers(-900, 900, (20, 64)) / 2.0])
    codes, scales = interpret.e4m3_rows(x)
    e = scales.astype(int) - 127
    top = np.abs(x).reshape(60, 2, 32).max(-1)
    assert (top <= 448 * 2.0 ** e).all() and (top > 448 * 2.0 ** (e - 1)).all()
    y = (x.reshape(60, 2, 32) / 2.0 ** e[..., None]).reshape(60, 64)
    want = torch.from_numpy(y).to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(codes, want)  # x are short enough for fp32 to hold y
    held = interpret.e4m3_held(codes, scales)
    step = np.maximum(np.abs(x), np.repeat(2.0 ** (e - 6), 32, 1).reshape(60, 64))
    assert (np.abs(held - x) <= step * 2.0 ** -4).all()  # 3 bits of mantissa, half a step


def test_e4m3_rows_at_the_ends():
    x = np.zeros((6, 32))
    x[1, 3] = 448.0
    x[2, 3] = np.nextafter(448.0, 449)
    x[3, :3] = [np.nan, -np.inf, 1.0]
    x[4, 0] = 3.3e38
    x[5, 0] = -65504.0
    codes, scales = interpret.e4m3_rows(x)
    assert list(scales[:, 0].astype(int) - 127) == [-117, 0, 1, -8, 119, 8]
    held = interpret.e4m3_held(codes, scales)
    assert held[1, 3] == 448 and held[2, 3] == 448 and not codes[0].any()
    assert np.isnan(held[3, :2]).all() and held[3, 2] == 1.0 and held[4, 0] == 448 * 2.0 ** 119
    codes, scales = interpret.e4m3_rows(x, fp16=True)
    assert interpret.e4m3_held(codes, scales)[5, 0] == -448 * 128.0  # finite in fp16


@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 3)])
def test_paged_attention_against_torch(causal, window):
    r = _rng(3)
    B, S, H, KV, D, N = 3, 4, 6, 2, 8, 12
    q, k, v = r.standard_normal((B, S, H, D)), r.standard_normal((B, N, KV, D)), r.standard_normal((B, N, KV, D))
    lengths, counts = [12, 7, 2], [4, 2, 4]
    o, lse, there = interpret.paged_attention(q, k, v, lengths, counts, causal, window)
    for b in range(B):
        n, L = counts[b], lengths[b]
        for j in range(S):
            if j >= n:
                assert not there[b, j]
                continue
            p = L - n + j
            mask = np.array([(not causal or i <= p) and (not window or i > p - window) for i in range(L)], bool)
            if not mask.any():
                assert not o[b, j].any() and np.isneginf(lse[b, j]).all()
                continue
            kk, vv = (torch.from_numpy(np.repeat(x[b, :L], H // KV, 1)).transpose(0, 1) for x in (k, v))
            want = torch.nn.functional.scaled_dot_product_attention(
                torch.from_numpy(q[b, j])[:, None], kk, vv, attn_mask=torch.from_numpy(mask)[None, None].expand(H, 1, L))
            assert np.allclose(o[b, j], want[:, 0].numpy(), atol=1e-13)
    assert not there[1, 2:].any() and there[0].all()
