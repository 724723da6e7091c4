"""The paged cache's operators and rotary positions, as a serving or training program uses them.

A decoder's step rotates its queries and keys, writes the new keys and values into a cache held in
pages, and attends over those pages; a program that goes on with a long prompt reads the cache back
as dense arrays.  ``listed`` names the cases, ``draw`` makes more of the same ranges, ``prepare`` makes
a case's inputs and handles, ``run`` is one pass (the framework's operators where ``own`` is true, else
elementary torch operations), ``exact`` the same results in float64.

Arrays are the library's column-major layouts, so a torch tensor holding one has the reversed
shape: (d, heads, positions, batch) is a (B, S, H, D) tensor here, and a cache's
(d, heads, positions in a page, pages) a (pages, page, KV, D) one, or (pages, KV, page, D) where the
heads lie outside the positions.
"""
from __future__ import annotations

import functools
import math
import sys

import torch

own = False

F32, BF16, F16, F64, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float64, torch.float8_e4m3fn
TYPES = {"f32": F32, "bf16": BF16, "f16": F16}


# ---- the cases -------------------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # A decoding step's queries and keys, one token a sequence, far into long texts: latency.
        {"name": "rotary_token", "kind": "rotary", "B": 16, "S": 1, "H": 32, "KV": 8, "D": 128, "R": 128, "axes": 1,
         "pairs": False, "dtype": "bf16", "gradient": False, "far": 1 << 20},
        # Training on video: time, height and width, the largest activations; memory-bound.
        {"name": "rotary_video", "kind": "rotary", "B": 8, "S": 4096, "H": 16, "KV": 16, "D": 128, "R": 128,
         "axes": 3, "pairs": False, "dtype": "bf16", "gradient": False, "far": 1024},
        # The gradient, fp32, on images: half the features rotated, adjacent pairs, a ragged length.
        {"name": "rotary_image_grad", "kind": "rotary", "B": 4, "S": 1023, "H": 12, "KV": 4, "D": 64, "R": 32,
         "axes": 2, "pairs": True, "dtype": "f32", "gradient": True, "far": 64},
        # A decoding step's new keys and values: one row a sequence and head into its page.
        {"name": "write_token", "kind": "write", "B": 16, "S": 1, "KV": 8, "D": 128, "cache": 4096, "page": 16,
         "outer": False, "dtype": "bf16", "e4m3": False, "ragged": False},
        # Prompts of several lengths, padded to the longest, fp16, pages of an odd size with the heads outside.
        {"name": "write_prompts", "kind": "write", "B": 4, "S": 1853, "KV": 4, "D": 64, "cache": 2400, "page": 24,
         "outer": True, "dtype": "f16", "e4m3": False, "ragged": True},
        # A prompt's next piece into an 8-bit cache, then the whole context read back for dense attention.
        {"name": "store_prompts_e4m3", "kind": "store", "B": 4, "S": 2048, "KV": 8, "D": 128, "cache": 8192,
         "page": 64, "outer": False, "dtype": "bf16", "e4m3": True, "ragged": True},
        # A large 8-bit cache read back.
        {"name": "read_contexts_e4m3", "kind": "read", "B": 8, "S": 1, "KV": 8, "D": 128, "cache": 16384, "page": 16,
         "outer": False, "dtype": "bf16", "e4m3": True, "ragged": False},
        # One short conversation: latency.
        {"name": "paged_short", "kind": "paged", "B": 1, "S": 1, "H": 32, "KV": 8, "D": 128, "cache": 600, "page": 16,
         "outer": False, "dtype": "bf16", "e4m3": False, "ragged": False, "window": 0},
        # A batch being served, sequences at every stage.
        {"name": "paged_batch", "kind": "paged", "B": 16, "S": 1, "H": 32, "KV": 8, "D": 128, "cache": 4096,
         "page": 16, "outer": False, "dtype": "bf16", "e4m3": False, "ragged": False, "window": 0},
        # Long contexts in 8 bits: the largest cache.
        {"name": "paged_long_e4m3", "kind": "paged", "B": 8, "S": 1, "H": 32, "KV": 8, "D": 128, "cache": 65536,
         "page": 64, "outer": False, "dtype": "bf16", "e4m3": True, "ragged": False, "window": 0},
        # Up to four proposed tokens a sequence checked at once, a sliding window, fp16, pages of seven.
        {"name": "paged_proposed_window", "kind": "paged", "B": 12, "S": 4, "H": 12, "KV": 4, "D": 64, "cache": 5000,
         "page": 7, "outer": False, "dtype": "f16", "e4m3": False, "ragged": True, "window": 1000},
        # One key/value head for all queries, 256 features, few long sequences: the split along the cache.
        {"name": "paged_one_head_d256", "kind": "paged", "B": 2, "S": 1, "H": 8, "KV": 1, "D": 256, "cache": 32768,
         "page": 32, "outer": True, "dtype": "bf16", "e4m3": False, "ragged": False, "window": 0},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "rotary", "write", "store", "read", "paged", "paged", "paged", "paged"])
    if kind == "rotary":
        kv, group, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4]), rng.choice([64, 80, 96, 128, 256])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        s = rng.choice([1, _log(rng, 2, 4096), _log(rng, 2, 4096)])
        most = (1 << 26) // (kv * (group + 1) * d * s)  # elements of q and k
        return {"kind": kind, "B": rng.randint(1, max(1, min(32, most))), "S": s, "H": kv * group, "KV": kv, "D": d,
                "R": rng.choice([d, d, d // 2, d // 4]), "axes": rng.choice([1, 1, 2, 3]),
                "pairs": rng.random() < 0.4, "dtype": dtype, "gradient": rng.random() < 0.4,
                "far": _log(rng, 16, 1 << 20)}
    kv, d, e4m3 = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256]), rng.random() < 0.5
    c = {"kind": kind, "KV": kv, "D": d, "page": rng.choice([1, 5, 16, 16, 24, 32, 64, 64, 128, 256]),
         "outer": rng.random() < 0.3, "dtype": rng.choice(["bf16", "bf16", "f16"]),
         "e4m3": kind != "write" and (e4m3 or kind == "store"), "ragged": rng.random() < 0.5}
    if kind == "paged":
        c["cache"] = _log(rng, 64, 65536)
        b = max(1, min(64, (1 << 27) // (kv * d * c["cache"])))
        c |= {"B": _log(rng, 1, b), "S": rng.choice([1, 1, 1, 2, 4, 8]), "H": kv * rng.choice([1, 2, 4, 4, 6, 8]),
              "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)])}
        return c
    c["cache"] = _log(rng, 64, 16384)
    b = max(1, min(32, (1 << 26) // (kv * d * c["cache"])))
    return c | {"B": _log(rng, 1, b), "S": 1 if kind == "read" else rng.choice([1, _log(rng, 2, c["cache"])])}


# ---- inputs ----------------------------------------------------------------------------

def _sections(c: dict) -> list[int]:
    """How many of the R / 2 pairs turn with each axis: time takes a quarter of them, space the rest."""
    n = c["R"] // 2
    return {1: [n], 2: [n // 2, n - n // 2], 3: [n // 4, (n - n // 4) // 2, n - n // 4 - (n - n // 4) // 2]}[c["axes"]]


def _positions(c: dict, gen: torch.Generator) -> torch.Tensor:
    """(B, S, axes) int32: a text's running position; an image's rows and columns, or a film's frames
    of 24 x 32 with them, from a place of each sequence's own."""
    at = torch.randint(0, c["far"], (c["B"], 1, c["axes"]), generator=gen)
    s = torch.arange(c["S"])
    own_axis = {1: [s], 2: [s // 32, s % 32], 3: [s // 768, s // 32 % 24, s % 32]}[c["axes"]]
    return (at + torch.stack(own_axis, -1)).to(torch.int32)


def _quantise(x: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes of x and, for each 32 features, the byte e of their scale 2^(e - 127): the least
    that brings the largest to 448 or less, so that dividing is exact and each value is rounded once.
    At least 2^-117 (every value the codes stand for is a normal number) and so small that
    448 times it is finite in x's type; larger values saturate."""
    f = x.float().unflatten(-1, (-1, 32))
    mantissa, exponent = torch.frexp(f.abs().amax(-1))       # mantissa in [1/2, 1)
    e = exponent - 9 + (mantissa > 0.875)                     # 448 = 0.875 * 2^9
    e = torch.where(mantissa == 0, -117, e).clamp(-117, 7 if dtype == F16 else 119)
    codes = torch.ldexp(f, -e[..., None]).clamp(-448, 448).to(E4M3)
    return codes.flatten(-2), (e + 127).to(torch.uint8)


def _in_pages(x: torch.Tensor, c: dict) -> torch.Tensor:
    """(pages, page, KV, n) in the case's order of memory."""
    return x.transpose(1, 2).contiguous() if c["outer"] else x


def _inputs(c: dict, seed: int) -> dict:
    gen = torch.Generator().manual_seed(int(seed) % (1 << 62))
    dgen = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62) + 1)

    def r(*shape):
        return torch.randn(*shape, device="cuda", generator=dgen)
    dt = TYPES[c["dtype"]]
    B, S, KV, D = c["B"], c["S"], c["KV"], c["D"]
    if c["kind"] == "rotary":
        theta = 10000.0 ** (-2.0 * torch.arange(c["R"] // 2, dtype=F64) / c["R"])
        return {"q": r(B, S, c["H"], D).to(dt), "k": r(B, S, KV, D).to(dt),
                "positions": _positions(c, gen).cuda(), "freqs": theta.to(F32).cuda()}
    # A cache of `cache` positions a sequence in pages of its own, in random order, and one page more, where
    # padding may be written; entries past a sequence's length name no page.
    width = -(-c["cache"] // c["page"])
    pages = B * width
    low = max(S, c["cache"] // 8)
    lengths = torch.randint(min(low, c["cache"]), c["cache"] + 1, (B,), generator=gen, dtype=torch.int32)
    lengths[int(torch.randint(0, B, (1,), generator=gen))] = c["cache"]
    table = torch.randperm(pages, generator=gen).to(torch.int32).view(B, width)
    table[torch.arange(width)[None, :] * c["page"] >= lengths[:, None]] = -1
    counts = torch.randint(1, S + 1, (B,), generator=gen, dtype=torch.int32) if c["ragged"] else None
    i = {"lengths": lengths.cuda(), "table": table.cuda(), "counts": None if counts is None else counts.cuda()}
    for name in ("k", "v"):
        held = r(pages + 1, c["page"], KV, D).to(dt)
        if c["e4m3"]:
            codes, scales = _quantise(held, dt)
            i[name + "_cache"], i[name + "_scales"] = _in_pages(codes, c), _in_pages(scales, c)
        else:
            i[name + "_cache"] = _in_pages(held, c)
        del held
        if c["kind"] in ("write", "store"):
            i[name] = r(B, S, KV, D).to(dt)
        if c["kind"] in ("store", "read"):
            i[name + "_dense"] = torch.zeros(B, c["cache"], KV, D, device="cuda", dtype=dt)
    if c["kind"] == "paged":
        i["q"] = r(B, S, c["H"], D).to(dt)
        i["o"] = torch.zeros_like(i["q"])
        i["lse"] = torch.zeros(B, S, c["H"], device="cuda")
    return i


def prepare(case: dict, seed: int) -> dict:
    state = {"case": case, **_inputs(case, seed)}
    if own:
        state |= _launches(case, state)
    return state


# ---- the framework's operators -----------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _framework():
    sys.path[:0] = ["tempest.jl_amd"]  # the package's folder, from the repository's root
    import tempest_hip as th
    import tempest_hip.launch as L
    return L, th.HIPTarget()


def _launches(c: dict, s: dict) -> dict:
    """The launches a program builds once for arrays that it keeps."""
    L, _ = _framework()
    B, S, KV, D = c["B"], c["S"], c["KV"], c["D"]
    dtype = {"f32": L.F32, "bf16": L.BF16, "f16": L.F16}[c["dtype"]]
    p = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
    if c["kind"] == "rotary":
        out = [torch.empty_like(s["q"]), torch.empty_like(s["k"])]
        return {"launches": [L.rotary(B, S, c["H"], KV, D, p["q"], p["k"], out[0].data_ptr(), out[1].data_ptr(),
                                      p["positions"], p["freqs"], sections=_sections(c), rotary_dim=c["R"],
                                      pairs=c["pairs"], inverse=c["gradient"], dtype=dtype)], "outputs": out}
    pages, page, width = s["k_cache"].shape[0] - 1, c["page"], s["table"].shape[1]
    cache = L.Cache(p["k_cache"], p["v_cache"], KV, D, page, pages, dtype=L.E4M3 if c["e4m3"] else dtype,
                    k_scales=p.get("k_scales", 0), v_scales=p.get("v_scales", 0),
                    strides=(page * D, D, KV * page * D) if c["outer"] else (D, KV * D, page * KV * D))
    if c["kind"] == "paged":
        launch = L.attention_paged(cache, B, c["H"], S, p["q"], p["o"], p["table"], p["lengths"], width,
                                   lse=p["lse"], counts=p.get("counts", 0), window=c["window"], dtype=dtype)
        return {"launches": [launch], "outputs": [s["o"], s["lse"]]}
    launches, outputs = [], []
    if c["kind"] in ("write", "store"):
        launches.append(L.cache_write(cache, B, S, p["k"], p["v"], p["table"], p["lengths"], width,
                                      counts=p.get("counts", 0), dtype=dtype))
        outputs = [s["k_cache"][:pages], s["v_cache"][:pages]]
    if c["kind"] in ("store", "read"):
        launches.append(L.cache_read(cache, B, c["cache"], p["k_dense"], p["v_dense"], p["table"], p["lengths"],
                                     width, dtype=dtype))
        outputs = [s["k_dense"], s["v_dense"]]
    return {"launches": launches, "outputs": outputs}


# ---- the plain forms ---------------------------------------------------------------------

def _angles(c: dict, s: dict) -> torch.Tensor:
    """(B, S, 1, R / 2), in 64 bits: positions far along a text are many turns."""
    n = _sections(c)
    by_pair = torch.cat([s["positions"][..., a:a + 1].expand(-1, -1, n[a]) for a in range(c["axes"])], -1)
    return (by_pair.double() * s["freqs"].double())[:, :, None, :]


def _rotary(c: dict, s: dict):
    angle = _angles(c, s)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    sin = -sin if c["gradient"] else sin
    R, out = c["R"], []
    for x in (s["q"], s["k"]):
        f = x.float()
        a, b = (f[..., 0:R:2], f[..., 1:R:2]) if c["pairs"] else (f[..., :R // 2], f[..., R // 2:R])
        u, v = a * cos - b * sin, a * sin + b * cos
        turned = torch.stack([u, v], -1).flatten(-2) if c["pairs"] else torch.cat([u, v], -1)
        out.append(torch.cat([turned, f[..., R:]], -1).to(x.dtype))
    return out


def _slots(c: dict, s: dict, positions: torch.Tensor):
    """Page and place in it of each position (B, n)."""
    return s["table"].long().gather(1, positions // c["page"]), positions % c["page"]


def _by_page(x: torch.Tensor, c: dict) -> torch.Tensor:
    return x.transpose(1, 2) if c["outer"] else x


def _write(c: dict, s: dict) -> None:
    B, S = c["B"], c["S"]
    counts = s["counts"].long() if s["counts"] is not None else torch.full((B,), S, device="cuda")
    j = torch.arange(S, device="cuda")
    at = (s["lengths"].long() - counts)[:, None] + j
    fits = (j < counts[:, None]) & (at >= 0)
    page, place = _slots(c, s, at.clamp(0, c["cache"] - 1))
    page = torch.where(fits, page, s["k_cache"].shape[0] - 1)  # padding to the page behind the last
    for n in ("k", "v"):
        if c["e4m3"]:
            codes, scales = _quantise(s[n], s[n].dtype)
            _by_page(s[n + "_cache"].view(torch.uint8), c)[page, place] = codes.view(torch.uint8)
            _by_page(s[n + "_scales"], c)[page, place] = scales
        else:
            _by_page(s[n + "_cache"], c)[page, place] = s[n]


def _gather(c: dict, s: dict, name: str) -> torch.Tensor:
    """The cache's first `cache` positions of every sequence, (B, cache, KV, D) in fp32."""
    at = torch.arange(c["cache"], device="cuda").expand(c["B"], -1)
    page, place = _slots(c, s, at)
    page = page.clamp(min=0)
    if not c["e4m3"]:
        return _by_page(s[name + "_cache"], c)[page, place].float()
    codes = _by_page(s[name + "_cache"].view(torch.uint8), c)[page, place].view(E4M3).float()
    scales = torch.exp2(_by_page(s[name + "_scales"], c)[page, place].float() - 127)
    return (codes.unflatten(-1, (-1, 32)) * scales[..., None]).flatten(-2)


def _read(c: dict, s: dict):
    held = (torch.arange(c["cache"], device="cuda") < s["lengths"][:, None])[..., None, None]
    return [torch.where(held, _gather(c, s, n).to(s[n + "_dense"].dtype), s[n + "_dense"]) for n in ("k", "v")]


def _seen(c: dict, s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Which keys each query sees, (B, S, cache), and which queries there are, (B, S)."""
    S = c["S"]
    counts = s["counts"][:, None] if s["counts"] is not None else S
    j = torch.arange(S, device="cuda")
    at = (s["lengths"][:, None] - counts + j)[..., None]
    key = torch.arange(c["cache"], device="cuda")
    seen = (key <= at) & (key < s["lengths"][:, None, None])
    return seen & (key > at - c["window"]) if c["window"] else seen, (j < counts).expand(c["B"], S)


def _paged(c: dict, s: dict):
    B, S, H, KV, D = c["B"], c["S"], c["H"], c["KV"], c["D"]
    seen, there = _seen(c, s)
    seen = seen.repeat_interleave(H // KV, 1)[:, None]                          # (B, 1, S group, cache)
    k = _gather(c, s, "k").permute(0, 2, 3, 1)                                  # (B, KV, D, cache)
    q = s["q"].float().view(B, S, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(B, KV, S * (H // KV), D)
    score = torch.matmul(q * (1.0 / math.sqrt(D)), k).masked_fill(~seen, -math.inf)
    del k
    top = score.amax(-1, keepdim=True)
    shift = torch.where(top == -math.inf, 0.0, top)
    weight = torch.exp(score - shift)
    total = weight.sum(-1, keepdim=True)
    o = torch.matmul(weight, _gather(c, s, "v").permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    lse = (shift + torch.log(total))[..., 0]
    o = o.view(B, KV, S, H // KV, D).permute(0, 2, 1, 3, 4).reshape(B, S, H, D).to(s["q"].dtype)
    lse = lse.view(B, KV, S, H // KV).permute(0, 2, 1, 3).reshape(B, S, H)
    return [torch.where(there[..., None, None], o, s["o"]), torch.where(there[..., None], lse, s["lse"])]


def run(state: dict):
    if own:
        for launch in state["launches"]:
            launch()
        return state["outputs"]
    c = state["case"]
    if c["kind"] == "rotary":
        return _rotary(c, state)
    if c["kind"] == "paged":
        return _paged(c, state)
    if c["kind"] in ("write", "store"):
        _write(c, state)
    if c["kind"] == "write":
        return [state["k_cache"][:-1], state["v_cache"][:-1]]
    return _read(c, state)


# ---- what a pass cannot do without -----------------------------------------------------

def work(case: dict) -> dict:
    c, e = case, 4 if case["dtype"] == "f32" else 2
    B, S, KV, D = c["B"], c["S"], c["KV"], c["D"]
    if c["kind"] == "rotary":
        n = B * S * (c["H"] + KV)
        return {"bytes": 2 * e * n * D + 4 * B * S * c["axes"] + 2 * c["R"], "flops": 3 * n * c["R"]}
    held = B * c["cache"] * 9 / 16                      # lengths spread evenly over 1/8..1 of the cache
    new = B * S * (0.5 if c["ragged"] else 1)
    row = KV * D * (33 / 32 if c["e4m3"] else e)        # a position of K, or of V
    if c["kind"] == "paged":
        mean = held / B if not c["window"] else min(held / B, c["window"])
        return {"bytes": 2 * B * mean * row + 2 * e * new * c["H"] * D,
                "flops": 4 * new * mean * c["H"] * D}
    wrote = 2 * new * (e * KV * D + row) if c["kind"] != "read" else 0
    read = 2 * held * (row + e * KV * D) if c["kind"] != "write" else 0
    moved = (new if c["kind"] != "read" else 0) + (held if c["kind"] != "write" else 0)
    return {"bytes": wrote + read, "flops": 2 * moved * KV * D}


# ---- the same in float64 ---------------------------------------------------------------

def _rotary_exact(c: dict, i: dict):
    """Each pair as a complex number, times e^(+-i theta)."""
    R, n = c["R"], _sections(c)
    axis = torch.tensor([a for a in range(c["axes"]) for _ in range(n[a])], device="cuda")
    theta = i["positions"].double()[..., axis] * i["freqs"].double()
    turn = torch.polar(torch.ones_like(theta), -theta if c["gradient"] else theta)[:, :, None]
    first = torch.arange(R // 2, device="cuda") * (2 if c["pairs"] else 1)
    second = first + (1 if c["pairs"] else R // 2)
    out = []
    for x in (i["q"].double(), i["k"].double()):
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        out.append(x)
    return out


def _rounded(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The values that e4m3 codes of x with a scale for each 32 features stand for, from the grid's
    definition: steps of 2^-3 of each power of two down to 2^-6, even below, ties to even."""
    y = x.double().unflatten(-1, (-1, 32))
    top = y.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -117)
    for k in range(-117, 8 if dtype == F16 else 120):
        e = torch.where(top > 448 * 2.0 ** (k - 1), max(k, -117), e)
    scale = torch.exp2(e)
    y = (y / scale).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step * scale).flatten(-2)


def _held(c: dict, i: dict, name: str, b: int, n: int) -> torch.Tensor:
    """Sequence b's first n positions as the cache holds them, (n, KV, D) in fp64."""
    at = torch.arange(n, device="cuda")
    page, place = i["table"][b].long()[at // c["page"]], at % c["page"]
    pick = (lambda x: x[page, :, place]) if c["outer"] else (lambda x: x[page, place])
    x = pick(i[name + "_cache"].view(torch.uint8)).view(E4M3).double() if c["e4m3"] else pick(i[name + "_cache"]).double()
    if c["e4m3"]:
        x *= torch.pow(2.0, pick(i[name + "_scales"]).double() - 127).repeat_interleave(32, -1)
    return x


def _stored(c: dict, i: dict, name: str, dense: bool):
    """The cache's arrays with the new rows in them, or what the sequences then hold."""
    caches = i[name + "_cache"][:-1].double() if not dense else None
    out = i[name + "_dense"].double() if dense else None
    for b in range(c["B"]):
        length = int(i["lengths"][b])
        new = 0 if c["kind"] == "read" else c["S"] if i["counts"] is None else int(i["counts"][b])
        if dense:
            out[b, :length] = _held(c, i, name, b, length)
        if new:
            x = _rounded(i[name][b, :new], i[name].dtype) if c["e4m3"] else i[name][b, :new].double()
            if dense:
                out[b, length - new:length] = x
            else:
                at = torch.arange(length - new, length, device="cuda")
                page, place = i["table"][b].long()[at // c["page"]], at % c["page"]
                if c["outer"]:
                    caches[page, :, place] = x
                else:
                    caches[page, place] = x
    return out if dense else caches


def _paged_exact(c: dict, i: dict):
    o, lse, group = i["o"].double(), i["lse"].double(), c["H"] // c["KV"]
    for b in range(c["B"]):
        length = int(i["lengths"][b])
        n = c["S"] if i["counts"] is None else int(i["counts"][b])
        k, v = (_held(c, i, x, b, length).transpose(0, 1) for x in ("k", "v"))
        for j in range(n):
            end = length - n + j + 1
            lo = max(0, end - c["window"]) if c["window"] else 0
            q = i["q"][b, j].double().view(c["KV"], group, c["D"])
            s = q @ k[:, lo:end].transpose(1, 2) / math.sqrt(c["D"])
            o[b, j] = (torch.softmax(s, -1) @ v[:, lo:end]).view(c["H"], c["D"])
            lse[b, j] = torch.logsumexp(s, -1).view(c["H"])
    return [o, lse]


def exact(case: dict, seed: int):
    c, i = case, _inputs(case, seed)
    if c["kind"] == "rotary":
        return _rotary_exact(c, i)
    if c["kind"] == "paged":
        return _paged_exact(c, i)
    return [_stored(c, i, n, c["kind"] != "write") for n in ("k", "v")]
