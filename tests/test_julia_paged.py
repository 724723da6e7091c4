"""The Julia extension's rotary positions and paged cache against the C ABI,
as test_julia_binding.py holds the rest: struct mirrors field by field and at gcc's
offsets, every builder reached, and each struct built with as many values as it has fields."""
import re

import pytest

import test_julia_binding as B

MIRRORS = {"RotaryDesc": "th_rotary_desc", "CCache": "th_cache", "CacheDesc": "th_cache_desc", "PagedDesc": "th_paged_desc"}


@pytest.fixture(autouse=True)
def _these(monkeypatch):
    monkeypatch.setattr(B, "MIRRORS", MIRRORS)


def test_mirrors_match_gcc_layout(tmp_path):
    B.test_struct_mirrors_match_gcc_layout(tmp_path)


def test_mirrors_cover_every_field():
    B.test_struct_mirrors_cover_every_c_field()


def test_every_builder_is_reached():
    used = {name for name, _, _ in B._ccalls()}
    assert {"th_build_rotary", "th_build_cache_write", "th_build_cache_read", "th_build_attention_paged"} <= used


@pytest.mark.parametrize("name", list(MIRRORS))
def test_structs_are_built_whole(name):
    fields = B._jl_structs()[name]
    built = [m for m in re.finditer(r"(?<!struct )(?<!\{)\b" + name + r"\(", B.JL)]
    assert built
    for m in built:
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, "[": 1, "{": 1, ")": -1, "]": -1, "}": -1}.get(B.JL[i], 0)
            i += 1
        args = B._split_top(B.JL[m.end():i - 1].replace("[", "(").replace("]", ")"))
        assert len(args) == len(fields), (name, len(args), len(fields))


# ---- what the wrappers refuse ------------------------------------------------
#
# No Julia runs here: each wrapper's `held(condition, message)` lines, and the one-line
# functions that they name, are read out of the text and evaluated over arrays that
# answer size, stride and eltype as Julia's do.

class Array:
    """A device array as the checks see it: column-major unless strides are given."""

    def __init__(self, eltype, *size, strides=None):
        self.eltype, self.size = eltype, size
        at, own = 1, []
        for n in size:
            own.append(at)
            at *= n
        self.strides = tuple(strides or own)


class Refused(Exception):
    pass


def _size(x, i=None):
    return x.size if i is None else x.size[i - 1] if i <= len(x.size) else 1


def _stride(x, i):
    return x.strides[i - 1] if i <= len(x.size) else sum(a * b for a, b in zip(x.strides, x.size))


def _prod(x):
    out = 1
    for n in x:
        out *= n
    return out


def _held(ok, what):
    if not ok:
        raise Refused(what)


def _python(e):
    """A Julia condition of the few forms the checks are written in."""
    e = re.sub(r"all\((\w+) -> (.*?), (\w+):(\w+\(\w+\)|\w+)\)(?=$|\s|\))",
               lambda m: f"all(({_python(m[2])}) for {m[1]} in range({m[3]}, {m[4]} + 1))", e)
    e = re.sub(r"\[1:\((\w+) - 1\)\]", r"[:\1 - 1]", e)
    for a, b in (("!==", " is not "), ("===", " is "), ("&&", " and "), ("||", " or "), ("nothing", "None")):
        e = e.replace(a, b)
    return e


def _block(start, text=None):
    """The body of the function that starts at the line `start`, up to its `end`."""
    text = B.JL if text is None else text
    at = text.index(start)
    indent = re.search(r"[ ]*$", text[:at])[0]
    return text[at:text.index("\n" + indent + "end\n", at)]


def _checks(body):
    """The checks of a body in order, as Python statements."""
    out = []
    for line in body.splitlines():
        line = line.strip()
        m = re.match(r'held\((.*), "(.*)"\)$', line)
        if m:
            out.append(f"_held({_python(m[1])}, {m[2]!r})")
        elif line.startswith("check_pages("):
            out.append(line)
        assert m or not line.startswith("held("), line
    return out


def _world():
    w = {"size": _size, "stride": _stride, "eltype": lambda x: x.eltype, "prod": _prod, "_held": _held,
         "length": lambda x: _prod(x.size) if isinstance(x, Array) else len(x), "ndims": lambda x: len(x.size),
         "UInt8": "UInt8", "Int32": "Int32", "Float32": "Float32"}
    for name in ("adjacent", "dense", "alike", "scales_fit", "integers"):
        m = re.search(rf"^{name}\((.*?)\) = ((?:.*&&\n)*.*)$", B.JL, flags=re.M)
        w[name] = eval(f"lambda {m[1]}: {_python(' '.join(m[2].split()))}", w)
    body = _checks(_block("function check_pages(table"))
    assert len(body) == 3
    exec("def check_pages(table, lengths, counts, batch):\n    " + "\n    ".join(body), w)
    return w


def _refusal(start, **args):
    """The message with which the function refuses its arguments, or None."""
    body = _checks(_block(start))
    assert body, start
    w = _world() | args
    try:
        for line in body:
            exec(line, w)
    except Refused as e:
        return str(e)


class _Cache:
    def __init__(self, k):
        self.k = k


HALF = "Float16"


def _rotary(**over):
    a = dict(q=Array(HALF, 64, 4, 5, 2), kk=Array(HALF, 64, 2, 5, 2), q_out=Array(HALF, 64, 4, 5, 2), ko=Array(HALF, 64, 2, 5, 2),
             positions=Array("Int32", 2, 5, 2), freqs=Array("Float32", 32), sections=(10, 22)) | over
    return _refusal("function rotary(", **a)


@pytest.mark.parametrize("over", [
    {}, dict(q_out=Array(HALF, 64, 4, 5, 2, strides=(1, 128, 512, 2560))),
    dict(q=Array(HALF, 64, 4, 5, 2, strides=(1, 64, 512, 2560))), dict(sections=(32,), positions=Array("Int32", 1, 5, 2))], ids=lambda o: ",".join(o) or "plain")
def test_rotary_takes(over):
    assert _rotary(**over) is None


@pytest.mark.parametrize("over", [
    dict(q=Array(HALF, 64, 4, 5, 2, strides=(2, 128, 512, 2560))), dict(q_out=Array("Float32", 64, 4, 5, 2)),
    dict(q_out=Array(HALF, 64, 4, 5, 1)), dict(kk=Array(HALF, 32, 2, 5, 2)), dict(ko=Array(HALF, 64, 1, 5, 2)),
    dict(kk=Array("Float32", 64, 2, 5, 2), ko=Array("Float32", 64, 2, 5, 2)), dict(kk=Array(HALF, 64, 2, 4, 2), ko=Array(HALF, 64, 2, 4, 2)),
    dict(positions=Array("Int64", 2, 5, 2)), dict(positions=Array("Int32", 2, 5, 1)), dict(positions=Array("Int32", 1, 5, 2)),
    dict(freqs=Array("Float64", 32)), dict(freqs=Array("Float32", 32, strides=(2,)))], ids=lambda o: ",".join(o))
def test_rotary_refuses(over):
    assert _rotary(**over)


def _paged(**over):
    a = dict(k=Array("UInt8", 64, 2, 16, 10), v=Array("UInt8", 64, 2, 16, 10), k_scales=Array("UInt8", 2, 2, 16, 10),
             v_scales=Array("UInt8", 2, 2, 16, 10)) | over
    return _refusal("function PagedCache(", **a)


OUTER = (1, 1024, 64, 2048)  # heads outside the positions


@pytest.mark.parametrize("over", [
    {}, dict(k=Array(HALF, 64, 2, 16, 10), v=Array(HALF, 64, 2, 16, 10), k_scales=None, v_scales=None),
    dict(k=Array("UInt8", 64, 2, 16, 10, strides=OUTER), v=Array("UInt8", 64, 2, 16, 10, strides=OUTER),
         k_scales=Array("UInt8", 2, 2, 16, 10, strides=(1, 32, 2, 64)), v_scales=Array("UInt8", 2, 2, 16, 10, strides=(1, 32, 2, 64)))], ids=lambda o: ",".join(o) or "plain")
def test_a_cache_takes(over):
    assert _paged(**over) is None


@pytest.mark.parametrize("over", [
    dict(v=Array("UInt8", 64, 2, 16, 10, strides=OUTER)), dict(v=Array("UInt8", 64, 2, 16, 9)), dict(v=Array(HALF, 64, 2, 16, 10)),
    dict(k=Array("UInt8", 64, 2, 16, 10, strides=(2, 128, 256, 4096))), dict(k_scales=None), dict(v_scales=None),
    dict(k_scales=Array("UInt8", 2, 2, 16, 10, strides=(1, 32, 2, 64))), dict(v_scales=Array("UInt8", 4, 2, 16, 10)),
    dict(v_scales=Array("Int32", 2, 2, 16, 10)), dict(k_scales=Array("UInt8", 2, 2, 16, 9))], ids=lambda o: ",".join(o))
def test_a_cache_refuses(over):
    assert _paged(**over)


PAGES = dict(table=Array("Int32", 7, 2), lengths=Array("Int32", 2), counts=None)
BAD_PAGES = [dict(table=Array("Int64", 7, 2)), dict(table=Array("Int32", 7, 3)), dict(table=Array("Int32", 7, 2, strides=(1, 8))),
             dict(table=Array("Int32", 7, 2, strides=(2, 1))), dict(lengths=Array("Int64", 2)), dict(lengths=Array("Int32", 1)),
             dict(lengths=Array("Int32", 2, strides=(2,))), dict(counts=Array("Int64", 2)), dict(counts=Array("Int32", 3))]


def _rows(**over):
    a = dict(c=_Cache(Array(HALF, 64, 2, 16, 10)), k=Array(HALF, 64, 2, 5, 2), v=Array(HALF, 64, 2, 5, 2)) | PAGES | over
    return _refusal("function cache_desc(", **a)


@pytest.mark.parametrize("over", [{}, dict(counts=Array("Int32", 2)), dict(k=Array(HALF, 64, 2, 5, 2, strides=(1, 320, 64, 640)),
                                                                           v=Array(HALF, 64, 2, 5, 2, strides=(1, 320, 64, 640)))], ids=lambda o: ",".join(o) or "plain")
def test_rows_taken(over):
    assert _rows(**over) is None


@pytest.mark.parametrize("over", [
    dict(v=Array(HALF, 64, 2, 5, 2, strides=(1, 320, 64, 640))), dict(v=Array(HALF, 64, 2, 4, 2)), dict(v=Array("BFloat16", 64, 2, 5, 2)),
    dict(k=Array(HALF, 32, 2, 5, 2), v=Array(HALF, 32, 2, 5, 2)), dict(k=Array(HALF, 64, 3, 5, 2), v=Array(HALF, 64, 3, 5, 2)),
    dict(k=Array(HALF, 64, 2, 5, 2, strides=(2, 128, 256, 1280))), *BAD_PAGES], ids=lambda o: ",".join(o))
def test_rows_refused(over):
    assert _rows(**over)


def _attention(**over):
    a = dict(cache=_Cache(Array(HALF, 64, 2, 16, 10)), q=Array(HALF, 64, 8, 3, 2), o=Array(HALF, 64, 8, 3, 2), lse=None) | PAGES | over
    return _refusal("function paged_attention(", **a)


@pytest.mark.parametrize("over", [{}, dict(lse=Array("Float32", 8, 3, 2), counts=Array("Int32", 2)),
                                  dict(q=Array(HALF, 64, 8, 1, 2, strides=(1, 64, 9, 512)), o=Array(HALF, 64, 8, 1, 2))], ids=lambda o: ",".join(o) or "plain")
def test_attention_takes(over):
    assert _attention(**over) is None


@pytest.mark.parametrize("over", [
    dict(o=Array(HALF, 64, 8, 3, 2, strides=(1, 192, 64, 1536))), dict(o=Array("Float32", 64, 8, 3, 2)), dict(o=Array(HALF, 64, 8, 2, 2)),
    dict(q=Array(HALF, 128, 8, 3, 2), o=Array(HALF, 128, 8, 3, 2)), dict(lse=Array(HALF, 8, 3, 2)), dict(lse=Array("Float32", 8, 3, 1)),
    dict(lse=Array("Float32", 8, 3, 2, strides=(6, 2, 1))), *BAD_PAGES], ids=lambda o: ",".join(o))
def test_attention_refuses(over):
    assert _attention(**over)


def test_launches_can_be_repointed():
    """Each launch has an operand for each of its values, under the number the header gives it."""
    for builder in ("th_build_rotary", "th_build_cache_write", "th_build_cache_read", "th_build_attention_paged"):
        at = B.JL.index(f"ccall((:{builder}, LIB)")
        n = int(re.search(r"by_value\((\d+)\)", B.JL[at:B.JL.index("\nend", at)])[1])
        doc = B.HEADER[:B.HEADER.index(f"int {builder}(")]
        doc = doc[doc.rindex("Values:"):]
        numbers = [int(x) for x in re.findall(r"(?:^|[,:*])\s*(\d+) ", doc.split("*/")[0])]
        if builder == "th_build_cache_read":
            assert "without counts" in doc and n == 8
        else:
            assert numbers == list(range(n)), (builder, numbers, n)
    assert "for i in 0:(n - 1)]" in _block("by_value(n) =", B.JL.replace("\n\n# What the library", "\nend\n\n# What the library"))
