"""What the rotary, cache and paged attention builders refuse, on the CPU: every
check comes before a device is asked for, so a descriptor that passes them all
ends in TH_E_STATE here.  And the page arithmetic, compiled for the host: quotients,
and table entries that name no page."""
import pathlib
import subprocess

import pytest
import torch

import tempest_hip.launch as L
from tempest_hip import HIPError

ROOT = pathlib.Path(__file__).resolve().parent.parent
ARGUMENT, STATE, UNSUPPORTED = -1, -2, -3
P = 1 << 20  # an address no check looks behind


@pytest.fixture(autouse=True)
def _no_device():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: valid descriptors would build")


def _code(f, *args, **kwargs):
    with pytest.raises(HIPError) as e:
        f(*args, **kwargs)
    return e.value.code


def _cache(**over):
    a = dict(k=P, v=P, heads=2, head_dim=64, page=16, pages=10, dtype=L.BF16) | over
    return L.Cache(**a)


E4M3 = dict(dtype=L.E4M3, k_scales=P, v_scales=P)


def _write(cache=None, **over):
    a = dict(batch=2, seq=3, k=P, v=P, table=P, lengths=P, table_pages=4) | over
    return L.cache_write(cache or _cache(), **a)


def _read(cache=None, **over):
    a = dict(batch=2, seq=3, k=P, v=P, table=P, lengths=P, table_pages=4) | over
    return L.cache_read(cache or _cache(), **a)


def _attend(cache=None, **over):
    a = dict(batch=2, heads=4, seq=1, q=P, o=P, table=P, lengths=P, table_pages=4) | over
    return L.attention_paged(cache or _cache(), **a)


BAD_CACHES = [dict(dtype=L.F32), dict(head_dim=60), dict(head_dim=264), dict(head_dim=0), dict(heads=0), dict(page=0),
              dict(pages=0), dict(page=1 << 16, pages=1 << 15), dict(k=0), dict(v=P + 8), dict(dtype=L.E4M3),
              dict(dtype=L.E4M3, k_scales=P, v_scales=P, head_dim=80), dict(dtype=L.E4M3, k_scales=P, v_scales=P + 2), dict(strides=(64, 100, 2048)),
              dict(strides=(64, -128, 2048)), dict(strides=(64, 64, 2048)), dict(strides=(64, 128, 1024)),
              dict(**E4M3, strides=(80, 160, 2560)), dict(strides=(64, 128, 1 << 61)), dict(strides=(1 << 62, 64, 2048))]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
@pytest.mark.parametrize("f", [_write, _read, _attend])
def test_a_cache_no_kernel_takes(f, bad):
    code = _code(f, _cache(**bad), **(dict(dtype=L.BF16) if bad.get("dtype") == L.F32 else {}))
    assert code == (UNSUPPORTED if bad.get("dtype") == L.F32 else ARGUMENT)


@pytest.mark.parametrize("good", [{}, dict(strides=(1024, 64, 2048)), dict(strides=(64, 256, 4096)), E4M3,
                                  dict(page=1, strides=(64, 0, 128)), dict(head_dim=8), dict(dtype=L.F16)], ids=str)
@pytest.mark.parametrize("f", [_write, _read, _attend])
def test_a_cache_every_kernel_takes(f, good):
    assert _code(f, _cache(**good)) == STATE


@pytest.mark.parametrize("f,bad", [
    (_write, dict(batch=0)), (_write, dict(batch=65536)), (_write, dict(seq=0)), (_write, dict(k=0)),
    (_write, dict(v=P + 1)), (_write, dict(table=0)), (_write, dict(lengths=0)), (_write, dict(table_pages=0)),
    (_write, dict(table_pages=1 << 27)), (_write, dict(counts=P + 2)), (_read, dict(table=P + 1)),
    (_attend, dict(lengths=P + 2)), (_attend, dict(lse=P + 2)), (_write, dict(strides=(-64, 128, 384))), (_write, dict(seq=1 << 28)),
    (_read, dict(strides=(64, 128, 256))), (_read, dict(strides=(32, 128, 384))), (_read, dict(k=0)),
    (_attend, dict(heads=3)), (_attend, dict(heads=0)), (_attend, dict(window=-1)),
    (_attend, dict(window=5, causal=False)), (_attend, dict(q=0)), (_attend, dict(o=P + 1)),
    (_attend, dict(q_strides=(64, 0, 128))), (_attend, dict(q_strides=(64, 256, -1))), (_attend, dict(table=0)),
    (_attend, dict(lengths=0)), (_attend, dict(seq=0)), (_attend, dict(batch=0)),
    (_attend, dict(seq=1 << 20, batch=1, q_strides=(64, 256, 0))), (_attend, dict(batch=65535, seq=200)),
    (_attend, dict(batch=64, table_pages=1 << 26))], ids=str)
def test_arguments_no_kernel_takes(f, bad):
    assert _code(f, **bad) == ARGUMENT


def test_the_largest_tables():
    assert _code(_attend, batch=32, table_pages=1 << 26) == STATE


@pytest.mark.parametrize("f", [_write, _read, _attend])
def test_types_that_do_not_go_together(f):
    assert _code(f, dtype=L.F16) == UNSUPPORTED
    assert _code(f, _cache(**E4M3), dtype=L.F32) == UNSUPPORTED
    assert _code(f, _cache(**E4M3), dtype=L.F16) == STATE


def test_reading_takes_no_counts():
    import ctypes
    from tempest_hip import _lib
    d = L._cache_desc(_cache(), 2, 3, P, P, P, P, 4, P, None, None)
    out = ctypes.c_void_p()
    assert _lib.load().th_build_cache_read(ctypes.byref(d), ctypes.byref(out)) == ARGUMENT


@pytest.mark.parametrize("name", ["rotary", "cache_write", "cache_read", "attention_paged"])
def test_null_descriptors(name):
    import ctypes
    from tempest_hip import _lib
    out = ctypes.c_void_p()
    assert getattr(_lib.load(), "th_build_" + name)(None, ctypes.byref(out)) == ARGUMENT


def _rotary(**over):
    a = dict(batch=2, seq=5, heads=4, kv_heads=2, head_dim=64, q=P, k=P, q_out=2 * P, k_out=2 * P, positions=P,
             freqs=P) | over
    return L.rotary(**a)


@pytest.mark.parametrize("bad", [
    dict(dtype=L.E4M3), dict(batch=0), dict(seq=0), dict(heads=0), dict(kv_heads=-1), dict(head_dim=0),
    dict(head_dim=2048), dict(rotary_dim=33), dict(rotary_dim=66), dict(sections=[]), dict(sections=[16, 8]),
    dict(sections=[40, -8]), dict(sections=[32, 1]), dict(positions=0), dict(freqs=0), dict(positions=P + 2), dict(q=0), dict(k_out=0),
    dict(q=P + 1), dict(dtype=L.F32, k=P + 2), dict(position_strides=(1, 1, -5)), dict(q_strides=(64, 256, -1)),
    dict(q_out_strides=(32, 256, 1280)), dict(k_out_strides=(64, 0, 640)),
    dict(q_out=P, q_strides=(64, 256, 1280), q_out_strides=(64, 512, 2560)), dict(batch=1 << 20, seq=1 << 20),
    dict(heads=65535)], ids=str)
def test_turns_no_kernel_takes(bad):
    assert _code(_rotary, **bad) == (UNSUPPORTED if bad.get("dtype") == L.E4M3 else ARGUMENT)


@pytest.mark.parametrize("good", [{}, dict(kv_heads=0, k=0, k_out=0), dict(rotary_dim=32, sections=[4, 6, 6]),
                                  dict(q_out=P, k_out=P), dict(position_strides=(0, 1, 0)), dict(dtype=L.F32),
                                  dict(q_strides=(0, 64, 0)), dict(sections=[0, 32])], ids=str)
def test_turns_every_kernel_takes(good):
    assert _code(_rotary, **good) == STATE


def test_more_axes_than_four():
    with pytest.raises(ValueError):
        _rotary(sections=[8, 8, 8, 4, 4])


def test_page_arithmetic_on_the_host(tmp_path):
    """cache.h's own functions: n / page for pages and positions across their range, and
    rows of entries that name no page, over a table of exactly its size."""
    src = tmp_path / "pages.hip"
    src.write_text(r'''
#include <cstdio>
#include <cstdlib>
#include "cache.h"
int main() {
  unsigned long long seed = 1;
  auto next = [&] { seed = seed * 6364136223846793005ull + 1442695040888963407ull; return (uint32_t)(seed >> 33); };
  for (int i = 0; i < 300000; ++i) {
    const int d = i < 4096 ? i + 1 : i < 4200 ? (1u << (i % 31)) + (i % 3) - 1 > 0 ? (int)((1u << (i % 31)) + (i % 3) - 1) : 1
                                              : (int)(next() >> (next() % 31)) | 1;
    const th::Divisor by = th::divisor(d);
    const int n[] = {0, 1, d - 1, d, (int)(next() >> 1), 0x7fffffff, (int)(0x7fffffffu / d * d), (int)(0x7fffffffu / d * d) - 1};
    for (int x : n)
      if (x >= 0 && thd::quotient(x, by) != x / d) return std::printf("%d / %d gave %d\n", x, d, thd::quotient(x, by)), 1;
  }
  int32_t* table = (int32_t*)std::malloc(6 * sizeof(int32_t));
  const int32_t entries[6] = {2, -1, 0, 3, 0x7fffffff, (int32_t)0x80000000};
  for (int i = 0; i < 6; ++i) table[i] = entries[i];
  const int32_t lengths[3] = {100, -5, 17}, counts[3] = {9, -1, 2};
  th_cache c{};
  c.page = 7, c.pages = 3, c.strides[0] = 8, c.strides[1] = 16, c.strides[2] = 200;
  const th::Pages p = th::pages_of(c, 2, table, lengths, counts);
  if (thd::length_of(p, 0) != 14 || thd::length_of(p, 1) != 0 || thd::length_of(p, 2) != 14) return 2;
  if (thd::count_of(p, 0, 4) != 4 || thd::count_of(p, 1, 4) != 0 || thd::count_of(p, 2, 4) != 2) return 3;
  for (int b = 0; b < 3; ++b)
    for (int at = 0; at < 14; ++at) {
      const int32_t e = entries[2 * b + at / 7];
      const int64_t want = e >= 0 && e < 3 ? e * 200 + at % 7 * 16 : -1;
      if (thd::row_of(p, b, at) != want) return 4;
    }
  std::puts("ok");
  return 0;
}
''')
    exe = tmp_path / "pages"
    csrc = ROOT / "tempest.jl_amd" / "csrc"
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-host-only", "-std=c++17", "-O1", "-I", str(csrc),
                    "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True, capture_output=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True)
    assert p.returncode == 0 and p.stdout == "ok\n", (p.returncode, p.stdout)
