"""The operators for drafted tokens without a GPU: parameter blocks against the C header's layout, the C
entries' refusals (before any CUDA call), the Python checks, and the oracle's own properties."""

import ctypes
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch

import draft_oracle as oracle
import fa
import fa.draft
import fa.pages
import fa.rotation
import tree_bound
from fa import _C

REPO = Path(__file__).resolve().parent.parent
CACHE = {"k": 16, "v": 32, "ks": 64, "vs": 128, "table": 4, "lengths": 4, "counts": 0, "k0": 4096, "k1": 1024, "v0": 4096, "v1": 1024,
         "ts": 3, "pages": 5, "page": 16, "most": 3, "hk": 2, "d": 64, "batch": 2, "tokens": 4, "cdtype": 2}


def _flat(f):
    return [x for v in f.values() for x in (v if isinstance(v, list) else [v])]


def _rotary(**kw):
    f = {"q": 16, "k": 16, "qo": 16, "ko": 16, "positions": 4, "cos": 16, "sin": 16, "strides": [64] * 6, "ps": [8, 4, 1], "batch": 1,
         "heads": 4, "hk": 2, "tokens": 4, "d": 64, "rotary": 64, "rows": 9, "axes": 2, "axis": bytes([1] * 32), "inter": 0, "inverse": 0,
         "dtype": 0} | kw
    return fa.rotation._PARAMS.pack(*_flat(f))


def _tree(**kw):
    f = CACHE | {"q": 16, "o": 16, "parents": 4, "strides": [64] * 3, "pstride": 4, "heads": 4, "window": 0, "sinks": 0, "scale": 0.1, "dtype": 0} | kw
    return fa.draft._TREE.pack(*_flat(f))


def _keep(**kw):
    f = CACHE | {"kept": 4, "new": 4, "kstride": 2, "n": 2} | kw
    return fa.draft._KEEP.pack(*_flat(f))


def _copy(**kw):
    f = CACHE | {"src": 4, "dst": 4, "n": 2} | kw
    return fa.pages._COPY.pack(*_flat(f))


def _pages(**kw):
    f = {"refs": 4, "table": 4, "from": 4, "rows": 4, "keep": 4, "lengths": 4, "counts": 0, "granted": 1, "src": 4, "dst": 4, "ts": 3,
         "fs": 3, "pages": 5, "batch": 2, "width": 3, "fb": 2, "tokens": 1, "page": 16} | kw
    return fa.pages._PAGES.pack(*_flat(f))


def test_packed_blocks_have_the_headers_layout(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text(r"""
#include <stdio.h>
#include "fa_b200.h"
#define P(x) printf("%lld ", (long long)(x))
static void cache(const FaCache* c) {
    P(c->k); P(c->v); P(c->k_scale); P(c->v_scale); P(c->page_table); P(c->lengths); P(c->counts);
    P(c->k_stride[0]); P(c->k_stride[1]); P(c->v_stride[0]); P(c->v_stride[1]); P(c->table_stride);
    P(c->num_pages); P(c->page_size); P(c->max_pages); P(c->kv_heads); P(c->head_dim); P(c->batch); P(c->tokens);
    P(c->dtype);
}
static void st(const int64_t* s) { P(s[0]); P(s[1]); P(s[2]); }
int main(int n, char** a) {
    FILE* f = fopen(a[1], "rb");
    FaRotaryParams r; FaTreeParams t; FaKeepParams k; FaCopyParams c; FaPages p;
    if (fread(&r, sizeof r, 1, f) != 1 || fread(&t, sizeof t, 1, f) != 1 || fread(&k, sizeof k, 1, f) != 1 ||
        fread(&c, sizeof c, 1, f) != 1 || fread(&p, sizeof p, 1, f) != 1) return 1;
    if (fgetc(f) != EOF) return 2;
    P(r.q); P(r.k); P(r.q_out); P(r.k_out); P(r.positions); P(r.cos); P(r.sin); st(r.q_stride); st(r.k_stride);
    st(r.position_stride); P(r.batch); P(r.heads); P(r.kv_heads); P(r.tokens); P(r.head_dim); P(r.rotary_dim);
    P(r.table_rows); P(r.axes); P(r.axis_of_pair[0]); P(r.axis_of_pair[63]); P(r.interleaved); P(r.inverse); P(r.dtype);
    printf("\n");
    cache(&t.cache); P(t.q); P(t.o); P(t.parents); st(t.q_stride); P(t.parent_stride); P(t.heads); P(t.window); P(t.sinks);
    P(t.softmax_scale); P(t.dtype); printf("\n");
    cache(&k.cache); P(k.kept); P(k.new_lengths); P(k.kept_stride); P(k.most); printf("\n");
    cache(&c.cache); P(c.src); P(c.dst); P(c.count); printf("\n");
    P(p.refs); P(p.table); P(p.from); P(p.rows); P(p.keep); P(p.lengths); P(p.counts); P(p.granted); P(p.src); P(p.dst);
    P(p.table_stride); P(p.from_stride); P(p.num_pages); P(p.batch); P(p.width); P(p.from_batch); P(p.tokens); P(p.page_size);
    return 0;
}
""")
    exe, data = tmp_path / "layout", tmp_path / "blocks"
    subprocess.run(["gcc", "-std=c99", "-w", "-I", str(REPO / "include"), "-o", str(exe), str(src)], check=True)
    axis = bytes([25]) + bytes(62) + bytes([26])
    numbers = list(range(1, 25)), list(range(27, 30))
    want, blob = [numbers[0] + [25, 26] + numbers[1]], fa.rotation._PARAMS.pack(*numbers[0], axis, *numbers[1])
    for block, count in ((fa.draft._TREE, 32), (fa.draft._KEEP, 24), (fa.pages._COPY, 23), (fa.pages._PAGES, 18)):
        values = list(range(1, count + 1))
        want.append(values)
        blob += block.pack(*values)
    data.write_bytes(blob)
    out = subprocess.run([str(exe), str(data)], capture_output=True, text=True, check=True).stdout
    assert [[int(x) for x in line.split()] for line in out.strip().splitlines()] == want


def _refused(entry, params, match, *rest):
    rc = getattr(_C.lib, entry)(params, *rest)
    message = _C.lib.fa_last_error().decode()
    assert rc == _C.FA_ERR_INVALID_ARGUMENT and re.search(match, message), message


@pytest.mark.parametrize("change,match", [
    ({"batch": 0}, "must be positive"), ({"heads": 0}, "must be positive"), ({"tokens": 0}, "must be positive"), ({"hk": 0}, "kv_heads with k"),
    ({"k": 0}, "kv_heads with k"), ({"batch": 65536}, "65535"), ({"tokens": (1 << 30) + 1}, "2\\^30"), ({"d": 96}, "head_dim"),
    ({"dtype": 2}, "dtype"), ({"q": 8}, "16-byte aligned"), ({"ko": 0}, "must be present"), ({"strides": [4] * 6}, "multiples of 8"),
    ({"rotary": 24}, "rotary_dim"), ({"rotary": 80}, "rotary_dim"), ({"rows": 0}, "rotary_dim"), ({"cos": 0}, "rotary_dim"),
    ({"axes": 0}, "1 to 4"), ({"axes": 5}, "1 to 4"), ({"axes": 1}, "axis_of_pair"), ({"positions": 0}, "positions"),
    ({"ps": [-1, 0, 0]}, "positions"),
])
def test_rotary_refusals(change, match):
    _refused("fa_rotary", _rotary(**change), match, None)


@pytest.mark.parametrize("change,match", [
    ({"batch": 0}, "must be positive"), ({"tokens": 0}, "must be positive"), ({"tokens": 257}, "at most 256"), ({"heads": 5}, "multiple of kv_heads"),
    ({"d": 80}, "head_dim"), ({"page": 12}, "power of two"), ({"cdtype": 1}, "tensors' type"), ({"ks": 0}, "scales"), ({"k": 8}, "16-byte aligned"),
    ({"window": -1}, "negative"), ({"sinks": -1}, "negative"), ({"window": 3}, "at least the number of nodes"), ({"scale": math.inf}, "finite"),
    ({"q": 0}, "must be present"), ({"o": 8}, "16-byte aligned"), ({"parents": 0}, "parents"), ({"pstride": -4}, "parents"), ({"dtype": 2}, "dtype"),
    ({"k0": 0}, "strides"), ({"v1": 0}, "strides"), ({"v0": 1 << 40}, "2\\^40"),
])
def test_tree_refusals(change, match):
    _refused("fa_tree_attention", _tree(**change), match, None, 0, None)
    _refused("fa_tree_workspace_size", _tree(**change), match, None)


@pytest.mark.parametrize("change,match", [
    ({"tokens": 257}, "at most 256"), ({"n": 5}, "at most the tokens"), ({"n": 0}, "at most the tokens"), ({"kept": 0}, "must be given"),
    ({"new": 0}, "must be given"), ({"kstride": -1}, "not negative"), ({"page": 7}, "power of two"), ({"cdtype": 3}, "dtype|type"),
])
def test_keep_refusals(change, match):
    _refused("fa_keep_tokens", _keep(**change), match, None)


@pytest.mark.parametrize("change,match", [
    ({"n": 0}, "must be positive"), ({"pages": 0}, "must be positive"), ({"hk": 0}, "must be positive"), ({"d": 96}, "head_dim"),
    ({"cdtype": 3}, "e4m3, float16"), ({"page": 4}, "power of two"), ({"vs": 0}, "scales"), ({"v1": 1032}, "multiples of 16"), ({"src": 0}, "src and dst"),
])
def test_copy_refusals(change, match):
    _refused("fa_copy_pages", _copy(**change), match, None)


@pytest.mark.parametrize("entries,change,match", [
    ("fork free reserve", {"batch": 0}, "must be positive"), ("fork free reserve", {"width": 0}, "must be positive"),
    ("fork free reserve", {"pages": 0}, "must be positive"), ("fork free reserve", {"batch": 65536}, "65535"),
    ("fork free reserve", {"ts": 2}, "a row apart"), ("fork free reserve", {"refs": 0}, "must be given"), ("fork free reserve", {"table": 0}, "must be given"),
    ("fork", {"from": 0}, "must be given"), ("fork", {"rows": 0}, "must be given"), ("fork", {"fb": 0}, "must be given"),
    ("reserve", {"page": 24}, "power of two"), ("reserve", {"tokens": 0}, "tokens"), ("reserve", {"width": 1 << 27, "ts": 1 << 27}, "2\\^31"),
    ("reserve", {"lengths": 0}, "must be given"), ("reserve", {"granted": 0}, "must be given"), ("reserve", {"dst": 0}, "must be given"),
])
def test_pages_refusals(entries, change, match):
    for entry in entries.split():
        if entry == "reserve":
            _refused("fa_reserve_workspace_size", _pages(**change), match, None)
            _refused("fa_reserve_pages", _pages(**change), match, None, 0, None)
        else:
            _refused(f"fa_{entry}_pages", _pages(**change), match, None)


def test_null_params_and_small_workspaces_are_refused():
    for entry, rest in (("fa_rotary", ()), ("fa_tree_attention", (None, 0)), ("fa_keep_tokens", ()), ("fa_copy_pages", ()),
                        ("fa_fork_pages", ()), ("fa_free_pages", ()), ("fa_reserve_pages", (None, 0))):
        _refused(entry, None, "NULL", *rest, None)
    for size, run, params in (("fa_tree_workspace_size", "fa_tree_attention", _tree()), ("fa_reserve_workspace_size", "fa_reserve_pages", _pages())):
        need = ctypes.c_uint64(0)
        assert getattr(_C.lib, size)(params, ctypes.byref(need)) == _C.FA_OK
        if need.value:
            for ptr, have in ((None, need.value), (16, need.value - 1), (24, need.value)):
                _refused(run, params, "workspace", ptr, have, None)


def test_python_checks_come_before_the_library():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    at, table = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(8, 32)
    for call in (fa.forward_rotary, fa.backward_rotary, fa.rotary):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(q, q, at, table, table)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.fork_pages(at[0], at, at[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.free_pages(at[0], at)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.reserve_pages(at[0], at, at[0], 1, 16)


def test_oracle_of_a_tree():
    #        0
    #      1   2      3 (on the context)
    #     4    5      6
    sees = oracle.ancestors([-1, 0, 0, -1, 1, 2, 3], 7)
    paths = [[0], [0, 1], [0, 2], [3], [0, 1, 4], [0, 2, 5], [3, 6]]
    assert [row.nonzero()[:, 0].tolist() for row in sees] == paths
    mask = oracle.tree_mask(torch.tensor([[-1, 0, 0]]), [5], [3], 6, 3, 0)[0]
    assert mask.int().tolist() == [[1, 1, 1, 0, 0, 0], [0, 1, 1, 1, 0, 0], [0, 1, 1, 0, 1, 0]]


def test_oracle_of_the_rotation_against_differences():
    """The inverse rotation is the gradient: against differences in 64 bits."""
    gen = torch.Generator().manual_seed(1)
    x, dy, step = (torch.randn(2, 3, 5, 64, generator=gen, dtype=torch.float64) for _ in range(3))
    positions = torch.randint(-1, 9, (3, 2, 5), generator=gen, dtype=torch.int32)
    angle = torch.rand(9, 24, generator=gen, dtype=torch.float64) * 6
    axes = [i % 3 for i in range(24)]
    for interleaved in (False, True):
        value = lambda h: (oracle.rotary(x + h * step, positions, angle.cos(), angle.sin(), axes, interleaved) * dy).sum()  # noqa: E731
        grad = oracle.rotary(dy, positions, angle.cos(), angle.sin(), axes, interleaved, inverse=True)
        h = 1e-4  # linear: no truncation, cancellation 1e-14 / h
        assert abs((value(h) - value(-h)) / (2 * h) - (grad * step).sum()) < 1e-8


def test_oracle_of_the_pages():
    pages = oracle.Pages([1, 0, 2, 0, 0])
    table = [[2, 0, -1], [2, -1, -1]]
    granted, src, dst = pages.reserve(table, [33, 9], 1, 16)
    # Row 0 needs its third page, row 1 shares its only one, which holds 8 older tokens.
    assert (granted, src, dst) == ([True, True], [-1, 2], [-1, 3]) and table == [[2, 0, 1], [3, -1, -1]]
    assert pages.refs == [1, 1, 1, 1, 0]
    fork = pages.fork(table, [1, -1, 0])
    assert fork == [[3, -1, -1], [-1, -1, -1], [2, 0, 1]] and pages.refs == [2, 2, 2, 2, 0]
    assert pages.reserve(table, [34, 10], 1, 16)[0] == [True, False]
    pages.free(fork, [1, 0, 0])
    assert fork == [[3, -1, -1], [-1, -1, -1], [-1, -1, -1]]


def test_the_derived_bound_by_hand():
    """Two keys, one a sink; what tree_bound allows is above the rounding of P and of the output and below twice their sum."""
    cache = type("Cache", (), dict(k=torch.zeros(1, 1, 8, 64), v=torch.ones(1, 1, 8, 64), k_scale=None, v_scale=None, num_pages=1, page_size=8, kv_heads=1))
    cache.k, cache.v = cache.k.half(), cache.v.half()
    cache.k[0, 0, 0] = 1.0
    cache.v[0, 0, 0] = 0.0
    q, lengths = torch.full((1, 1, 1, 64), 2.0, dtype=torch.float16), torch.tensor([2], dtype=torch.int32)
    o, bound = tree_bound.tree(q, cache, torch.tensor([[0]]), lengths, torch.tensor([[-1]]), scale=1 / 64)
    want = 1 / (1 + math.exp(2))
    assert abs(o[0, 0, 0, 0].item() - want) < 1e-12
    assert 2 * 2.0**-11 * want < bound[0, 0, 0, 0].item() < 4 * 2.0**-11 * want


def test_pools_beyond_the_kernels_indexes_are_refused():
    for entry in ("fork", "free"):
        _refused(f"fa_{entry}_pages", _pages(pages=(1 << 30) + 1), "num_pages", None)
    _refused("fa_reserve_workspace_size", _pages(pages=(1 << 30) + 1), "num_pages", None)
    _refused("fa_reserve_pages", _pages(pages=2**31 - 1), "num_pages", None, 0, None)
