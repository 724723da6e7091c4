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
