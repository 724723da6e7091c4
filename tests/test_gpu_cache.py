"""Writing a paged cache and reading it back, against the oracle: 16-bit rows
to the bit, e4m3 codes and scale bytes to the bit (the definition has one rounding,
to nearest even), what is read back from them exactly where the type holds it."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import interpret

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


class Paged:
    """A cache's arrays on the device, (pages, page, KV, D) views of them, a table."""

    def __init__(self, B, cap, KV, D, page, dtype="bf16", e4m3=False, outer=False, spare=2, seed=0):
        import tempest_hip.launch as L
        self.B, self.KV, self.D, self.page, self.dtype, self.e4m3 = B, KV, D, page, dtype, e4m3
        self.width = -(-cap // page)
        self.pages = B * self.width + spare
        gen = torch.Generator().manual_seed(seed)
        self.table = torch.randperm(self.pages, generator=gen)[:B * self.width].to(torch.int32).view(B, -1).cuda()
        held = torch.uint8 if e4m3 else TYPES[dtype]
        shape = (self.pages, KV, page) if outer else (self.pages, page, KV)
        fill = 0x2a if e4m3 else 5.0
        self.memory = [torch.full((*shape, D), fill, device="cuda", dtype=held) for _ in range(2)]
        self.scale_memory = [torch.full((*shape, D // 32), 120, device="cuda", dtype=torch.uint8) for _ in range(2)]
        turn = (lambda t: t.transpose(1, 2)) if outer else (lambda t: t)
        self.k, self.v = map(turn, self.memory)
        self.ks, self.vs = map(turn, self.scale_memory)
        dt = {"bf16": L.BF16, "f16": L.F16}[dtype]
        self.type = dt
        s = self.k.stride()
        extra = dict(k_scales=self.ks.data_ptr(), v_scales=self.vs.data_ptr()) if e4m3 else {}
        self.cache = L.Cache(self.k.data_ptr(), self.v.data_ptr(), KV, D, page, self.pages,
                             dtype=L.E4M3 if e4m3 else dt, strides=(s[2], s[1], s[0]), **extra)

    def where(self, b, at):
        return int(self.table[b, at // self.page]), at % self.page

    def held(self, array="k"):
        """(pages, page, KV, D) float64: what the arrays stand for."""
        t = getattr(self, array)
        if not self.e4m3:
            return t.double().cpu().numpy()
        return interpret.e4m3_held(t.cpu().numpy(), getattr(self, array + "s").cpu().numpy())

    def sequences(self, n, array="k"):
        """(B, n, KV, D): the positions in order (a page that is none: zeros)."""
        h, out = self.held(array), np.zeros((self.B, n, self.KV, self.D))
        table = self.table.cpu().numpy()
        for b in range(self.B):
            for at in range(min(n, self.width * self.page)):
                page = table[b, at // self.page]
                if 0 <= page < self.pages:
                    out[b, at] = h[page, at % self.page]
        return out


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def rows(gen, dtype, *shape, spread=True, offset=0):
    n = int(np.prod(shape))
    x = torch.randn(*shape, device="cuda", generator=gen)
    if spread:  # rows of many sizes, so that every scale and the steps below the least normal code occur
        x = x * torch.exp2(torch.randint(-12, 5, shape[:-1], device="cuda", generator=gen).float())[..., None]
        x = x * torch.exp2(-torch.randint(0, 14, shape, device="cuda", generator=gen).float())
    t = torch.empty(n + offset, device="cuda", dtype=TYPES[dtype])[offset:].view(*shape)
    return t.copy_(x)


CASES = [  # B, S, KV, D, page, cap, dtype, e4m3, outer, lengths, counts, offset
    (1, 1, 1, 8, 1, 1, "bf16", False, False, [1], None, 0),
    (3, 1, 8, 128, 16, 100, "bf16", False, False, [100, 1, 16], None, 0),
    (3, 1, 8, 128, 16, 100, "bf16", True, False, [17, 1, 100], None, 0),
    (2, 40, 3, 80, 7, 60, "f16", False, True, [50, 40], [40, 13], 1),
    (2, 40, 3, 96, 7, 60, "f16", True, True, [50, 40], [40, 13], 3),
    (4, 33, 2, 64, 24, 72, "bf16", True, False, [72, 33, 5, 0], [33, 0, 5, 3], 0),
    (4, 33, 2, 256, 64, 64, "bf16", True, True, [64, 40, 10, 33], [33, 1, 20, 33], 1),
    (2, 300, 4, 32, 128, 500, "f16", True, False, [400, 300], None, 0),
    (2, 5, 5, 248, 3, 20, "bf16", False, False, [400, -7], [9, 2], 0)]


@pytest.mark.parametrize("B,S,KV,D,page,cap,dtype,e4m3,outer,lengths,counts,offset", CASES)
def test_write_and_read(target, B, S, KV, D, page, cap, dtype, e4m3, outer, lengths, counts, offset):
    import tempest_hip.launch as L
    announce("cache", B, S, KV, D, page, cap, dtype, e4m3, outer, lengths, counts, offset)
    c = Paged(B, cap, KV, D, page, dtype, e4m3, outer)
    gen = torch.Generator(device="cuda").manual_seed(D + page)
    k, v = rows(gen, dtype, B, S, KV, D, offset=offset), rows(gen, dtype, B, S, KV, D, offset=offset)
    n, m = ints(*lengths), ints(*(counts or [S] * B))
    want = {x: (getattr(c, x).cpu().clone(), getattr(c, x + "s").cpu().clone()) for x in "kv"}
    total = c.width * page
    for name, new in (("k", k), ("v", v)):
        codes, scales = (interpret.e4m3_rows(new.double().cpu().numpy(), dtype == "f16") if e4m3 else (None, None))
        for b in range(B):
            length, count = min(max(lengths[b], 0), total), min(max(counts[b] if counts else S, 0), S)
            for j in range(count):
                if length - count + j >= 0:
                    at = c.where(b, length - count + j)
                    want[name][0][at] = torch.from_numpy(codes[b, j]) if e4m3 else new[b, j].cpu()
                    if e4m3:
                        want[name][1][at] = torch.from_numpy(scales[b, j])
    write = L.cache_write(c.cache, B, S, k.data_ptr(), v.data_ptr(), c.table.data_ptr(), n.data_ptr(), c.width,
                          counts=m.data_ptr() if counts else 0, dtype=c.type)
    for _ in range(2):  # writing the same again changes nothing
        write()
        torch.cuda.synchronize()
        for x in "kv":
            assert torch.equal(getattr(c, x).cpu(), want[x][0]), x
            assert not e4m3 or torch.equal(getattr(c, x + "s").cpu(), want[x][1]), x
    # Read back: held rows exactly, the others as they were.
    seq = total + 3
    out = [torch.full((B * seq * KV * D + offset,), -9.0, device="cuda", dtype=TYPES[dtype])[offset:].view(B, seq, KV, D)
           for _ in range(2)]
    L.cache_read(c.cache, B, seq, *(t.data_ptr() for t in out), c.table.data_ptr(), n.data_ptr(), c.width, dtype=c.type)()
    torch.cuda.synchronize()
    for x, t in zip("kv", out):
        ref = torch.from_numpy(c.sequences(seq, x)).to(TYPES[dtype])  # (rounded once: what e4m3 holds may be below fp16's normals)
        for b in range(B):
            length = min(max(lengths[b], 0), total)
            assert torch.equal(t[b, :length].cpu(), ref[b, :length]) and (t[b, length:] == -9.0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_every_code_and_scale(target, dtype):
    """Rows whose 32 features are one scale's codes, halves and quarters between them, at scales
    across the range; zeros, the type's largest and least values, NaN and infinities."""
    import tempest_hip.launch as L
    announce("cache codes", dtype)
    grid = interpret.e4m3_values()[:127]
    y = np.sort(np.concatenate([grid, (grid[1:] + grid[:-1]) / 2, grid[:-1] * 0.75 + grid[1:] * 0.25]))
    y = np.resize(np.concatenate([y, -y]), (26, 31))
    blocks = np.concatenate([np.full((26, 1), 448.0), y], 1)
    exponents = range(-14, 8) if dtype == "f16" else list(range(-117, 120, 13)) + [118, 119]
    x = torch.from_numpy(np.concatenate([blocks * 2.0 ** e for e in exponents] + [np.zeros((2, 32))])).to(TYPES[dtype])
    x[-1, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0])
    info = torch.finfo(TYPES[dtype])
    x[-2, :3] = torch.tensor([info.max, info.smallest_normal, info.min], dtype=TYPES[dtype])
    if dtype == "bf16":
        x = torch.cat([x, torch.full((1, 32), 2.0 ** -130, dtype=TYPES[dtype])])
    x = x.cuda().contiguous()
    n = x.shape[0]
    c = Paged(1, n, 1, 32, 8, dtype, True)
    out = [torch.empty_like(x) for _ in range(2)]
    length = ints(n)
    L.cache_write(c.cache, 1, n, x.data_ptr(), x.data_ptr(), c.table.data_ptr(), length.data_ptr(), c.width, dtype=c.type)()
    L.cache_read(c.cache, 1, n, *(t.data_ptr() for t in out), c.table.data_ptr(), length.data_ptr(), c.width, dtype=c.type)()
    torch.cuda.synchronize()
    codes, scales = interpret.e4m3_rows(x.double().cpu().numpy(), dtype == "f16")
    table = c.table.cpu()[0].long()
    got = c.k.cpu()[table].reshape(-1, 32)[:n].numpy()
    nan = codes & 127 == 127
    assert np.array_equal(c.ks.cpu()[table].reshape(-1, 1)[:n].numpy(), scales)
    assert np.array_equal(got[~nan], codes[~nan]) and (got[nan] & 127 == 127).all()
    want = torch.from_numpy(interpret.e4m3_held(codes, scales)).to(TYPES[dtype])
    for t in out:
        assert torch.equal(t.cpu().nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))
        assert torch.equal(t.cpu().isnan(), want.isnan())


@pytest.mark.parametrize("e4m3", [False, True])
def test_entries_that_name_no_page(target, e4m3):
    """Below 0, past the last page, far past it: nothing written, zeros read."""
    import tempest_hip.launch as L
    announce("cache bad pages", e4m3)
    B, S, KV, D, page = 2, 24, 2, 64, 8
    c = Paged(B, S, KV, D, page, "bf16", e4m3)
    c.table[0, 1], c.table[1, 0], c.table[1, 2] = -1, c.pages, 0x7fffffff
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = rows(gen, "bf16", B, S, KV, D), rows(gen, "bf16", B, S, KV, D)
    before = [t.clone() for t in c.memory + c.scale_memory]
    out = [torch.full((B, S, KV, D), -9.0, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    n = ints(S, S)
    L.cache_write(c.cache, B, S, k.data_ptr(), v.data_ptr(), c.table.data_ptr(), n.data_ptr(), c.width)()
    L.cache_read(c.cache, B, S, *(t.data_ptr() for t in out), c.table.data_ptr(), n.data_ptr(), c.width)()
    torch.cuda.synchronize()
    used = {int(c.table[b, i]) for b, i in ((0, 0), (0, 2), (1, 1))}
    for was, now in zip(before, c.memory + c.scale_memory):
        for page_ in range(c.pages):
            assert page_ in used or torch.equal(was[page_], now[page_])
    for x, t in zip("kv", out):
        assert torch.equal(t.double().cpu(), torch.from_numpy(c.sequences(S, x)))
    assert not out[0][0, 8:16].any() and not out[1][1, :8].any() and out[0][0, :8].any()


def test_a_recorded_write_follows_the_device(target):
    """Written and read token by token from one graph, lengths counted up on the device."""
    import tempest_hip.launch as L
    announce("cache graph")
    B, KV, D, page, steps = 3, 2, 64, 4, 10
    c = Paged(B, steps, KV, D, page, "bf16", False)
    gen = torch.Generator(device="cuda").manual_seed(4)
    k, v = rows(gen, "bf16", B, 1, KV, D), rows(gen, "bf16", B, 1, KV, D)
    out = [torch.zeros(B, steps, KV, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    n = ints(0, 0, 0)
    write = L.cache_write(c.cache, B, 1, k.data_ptr(), v.data_ptr(), c.table.data_ptr(), n.data_ptr(), c.width)
    read = L.cache_read(c.cache, B, steps, *(t.data_ptr() for t in out), c.table.data_ptr(), n.data_ptr(), c.width)
    graph = target.capture([write, read])
    want = torch.zeros_like(out[0])
    for i in range(steps):
        k.copy_(rows(gen, "bf16", B, 1, KV, D))
        n.add_(1)
        want[:, i] = k[:, 0]
        target.replay(graph)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want)


def test_a_cache_past_32_bits(target):
    """Pages whose elements lie past 2^32 of the arrays' start."""
    import tempest_hip.launch as L
    announce("cache past 2^32")
    KV, D, page, pages = 8, 256, 64, 34000  # 4.46e9 elements
    k = torch.empty(pages, page, KV, D, device="cuda", dtype=torch.uint8)
    ks = torch.empty(pages, page, KV, D // 32, device="cuda", dtype=torch.uint8)
    cache = L.Cache(k.data_ptr(), k.data_ptr(), KV, D, page, pages, dtype=L.E4M3, k_scales=ks.data_ptr(),
                    v_scales=ks.data_ptr())
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = rows(gen, "bf16", 1, 130, KV, D)
    table = ints(33999, 33000, 5)
    n = ints(130)
    out = torch.zeros_like(x)
    L.cache_write(cache, 1, 130, x.data_ptr(), x.data_ptr(), table.data_ptr(), n.data_ptr(), 3)()
    L.cache_read(cache, 1, 130, out.data_ptr(), out.data_ptr(), table.data_ptr(), n.data_ptr(), 3)()
    torch.cuda.synchronize()
    codes, scales = interpret.e4m3_rows(x.double().cpu().numpy())
    assert torch.equal(out.double().cpu(), torch.from_numpy(interpret.e4m3_held(codes, scales)))
    assert torch.equal(k[33999].cpu(), torch.from_numpy(codes[0, :64]))


@pytest.mark.parametrize("e4m3", [False, True])
def test_repointed_to_odd_elements(target, e4m3):
    """Dense rows at an odd element, given after the launch was built; the cache's arrays stay at 16 bytes."""
    import tempest_hip.launch as L
    from tempest_hip import HIPError
    announce("cache odd elements", e4m3)
    B, S, KV, D, page = 2, 11, 2, 64, 4
    c = Paged(B, S, KV, D, page, "bf16", e4m3)
    gen = torch.Generator(device="cuda").manual_seed(5)
    k, v = rows(gen, "bf16", B, S, KV, D), rows(gen, "bf16", B, S, KV, D)
    n = ints(S, S)
    write = L.cache_write(c.cache, B, S, k.data_ptr(), v.data_ptr(), c.table.data_ptr(), n.data_ptr(), c.width)
    read = L.cache_read(c.cache, B, S, k.data_ptr(), v.data_ptr(), c.table.data_ptr(), n.data_ptr(), c.width)
    k2, v2 = rows(gen, "bf16", B, S, KV, D, offset=1), rows(gen, "bf16", B, S, KV, D, offset=3)
    out = [torch.zeros(B * S * KV * D + 1, device="cuda", dtype=torch.bfloat16)[1:].view(B, S, KV, D) for _ in range(2)]
    write.repoint("k", k2.data_ptr())
    write.repoint("v", v2.data_ptr())
    read.repoint("k", out[0].data_ptr())
    read.repoint("v", out[1].data_ptr())
    write()
    read()
    torch.cuda.synchronize()
    for x, t in zip((k2, v2), out):
        want = x.double().cpu().numpy()
        if e4m3:
            want = interpret.e4m3_held(*interpret.e4m3_rows(want))
        assert torch.equal(t.double().cpu(), torch.from_numpy(want))
    with pytest.raises(HIPError):
        write.repoint("k", k2.data_ptr() + 1)
    with pytest.raises(HIPError):
        write.repoint("k_cache", c.k.data_ptr() + 8)
