"""The streaming operators without a GPU: their parameter blocks against the C header's layout, the
C entries' refusals (before any CUDA call), the Python checks, and the oracle's gradient against
differences in 64 bits."""

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

import fa
import fa.cache
import fa.window
import stream_oracle as oracle
from fa import _C

REPO = Path(__file__).resolve().parent.parent


def test_packed_blocks_have_the_headers_layout(tmp_path):
    """Every field gets a value of its own, packed as the binding packs it and printed by C."""
    src = tmp_path / "layout.c"
    src.write_text(r"""
#include <stdio.h>
#include <string.h>
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
    FaWindowParams w; FaAppendParams p; FaCachedParams c;
    if (fread(&w, sizeof w, 1, f) != 1 || fread(&p, sizeof p, 1, f) != 1 || fread(&c, sizeof c, 1, f) != 1) return 1;
    if (fgetc(f) != EOF) return 2;
    P(w.q); P(w.k); P(w.v); P(w.o); P(w.lse); P(w.d_o); P(w.dq); P(w.dk); P(w.dv);
    st(w.q_stride); st(w.k_stride); st(w.v_stride); st(w.o_stride); st(w.do_stride); st(w.dq_stride); st(w.dk_stride);
    st(w.dv_stride); P(w.batch); P(w.heads); P(w.kv_heads); P(w.q_len); P(w.k_len); P(w.head_dim); P(w.window);
    P(w.sinks); P(w.softmax_scale); P(w.dtype); printf("\n");
    cache(&p.cache); P(p.k_new); P(p.v_new); P(p.q); P(p.q_out); P(p.cos); P(p.sin); st(p.k_new_stride);
    st(p.v_new_stride); st(p.q_stride); P(p.heads); P(p.table_rows); P(p.rotary_dim); P(p.interleaved); P(p.dtype);
    printf("\n");
    cache(&c.cache); P(c.q); P(c.o); st(c.q_stride); P(c.heads); P(c.window); P(c.sinks); P(c.softmax_scale); P(c.dtype);
    return 0;
}
""")
    exe, data = tmp_path / "layout", tmp_path / "blocks"
    subprocess.run(["gcc", "-std=c99", "-w", "-I", str(REPO / "include"), "-o", str(exe), str(src)], check=True)
    want, blob = [], b""
    for block, count in ((fa.window._PARAMS, 43), (fa.cache._APPEND, 40), (fa.cache._CACHED, 30)):
        values = list(range(1, count + 1))
        want.append(values)
        blob += block.pack(*values)
    data.write_bytes(blob)
    out = subprocess.run([str(exe), str(data)], capture_output=True, text=True, check=True).stdout
    assert [[int(x) for x in line.split()] for line in out.strip().splitlines()] == want


def _call(entry, params, *rest):
    rc = getattr(_C.lib, entry)(params, *rest)
    return rc, _C.lib.fa_last_error().decode()


def _window(**kw):
    f = dict(zip("q k v o lse do dq dk dv".split(), (16 * (i + 1) for i in range(9))))
    f |= {"strides": [64 * 64, 64, 64] * 8, "batch": 1, "heads": 4, "kv_heads": 2, "q_len": 8, "k_len": 8, "head_dim": 64,
          "window": 4, "sinks": 1, "scale": 0.1, "dtype": 0}
    f |= kw
    return fa.window._PARAMS.pack(*(x for v in f.values() for x in (v if isinstance(v, list) else [v])))


@pytest.mark.parametrize("change,match", [
    ({"batch": 0}, "must be positive"), ({"q_len": -1}, "must be positive"), ({"k_len": 0}, "must be positive"),
    ({"heads": 3}, "multiple of kv_heads"), ({"head_dim": 96}, "head_dim"), ({"window": -1}, "negative"),
    ({"sinks": -1}, "negative"), ({"dtype": 2}, "dtype"), ({"scale": math.nan}, "finite"), ({"batch": 65536}, "65535"),
    ({"q": 0}, "must be present"), ({"k": 8}, "16-byte aligned"), ({"dv": 0}, "must be present"), ({"lse": 0}, "must be present"),
    ({"strides": [64 * 64, 64, 63] * 8}, "multiples of 8"), ({"strides": [64, 64, -64] * 8}, "multiples of 8"),
    ({"q_len": (1 << 30) + 1}, "2\\^30"), ({"strides": [0, 64, 64] * 8, "batch": 2}, "positive strides"),
    ({"strides": [64, 0, 64] * 8}, "positive strides"),
])
def test_window_refusals(change, match):
    import re

    for entry, rest in (("fa_window_bwd", (None, 0, None)), ("fa_window_bwd_workspace_size", (None,))):
        rc, message = _call(entry, _window(**change), *rest)
        assert rc == _C.FA_ERR_INVALID_ARGUMENT and re.search(match, message), message
    if not {"dv", "lse"} & change.keys():
        rc, message = _call("fa_window_fwd", _window(**change), None)
        assert rc == _C.FA_ERR_INVALID_ARGUMENT and re.search(match, message), message


def test_null_params_and_small_workspaces_are_refused():
    for entry, rest in (("fa_window_fwd", (None,)), ("fa_window_bwd", (None, 0, None)), ("fa_append_kv", (None,)),
                        ("fa_cached_attention", (None, 0, None))):
        rc, message = _call(entry, None, *rest)
        assert rc == _C.FA_ERR_INVALID_ARGUMENT and "NULL" in message
    need = ctypes.c_uint64(0)
    assert _C.lib.fa_window_bwd_workspace_size(_window(), ctypes.byref(need)) == _C.FA_OK and need.value > 0
    for ptr, size in ((None, need.value), (16, need.value - 1), (24, need.value)):
        rc, message = _call("fa_window_bwd", _window(), ptr, size, None)
        assert rc == _C.FA_ERR_INVALID_ARGUMENT and "workspace" in message


CACHE = {"k": 16, "v": 32, "ks": 64, "vs": 128, "table": 4, "lengths": 4, "counts": 0, "k0": 4096, "k1": 1024, "v0": 4096, "v1": 1024,
         "ts": 3, "pages": 5, "page": 16, "most": 3, "hk": 2, "d": 64, "batch": 2, "tokens": 1, "cdtype": 2}


def _append(**kw):
    f = CACHE | {"kn": 16, "vn": 16, "q": 16, "qo": 16, "cos": 16, "sin": 16, "strides": [64] * 9, "heads": 4, "rows": 9,
                 "rotary": 64, "inter": 0, "dtype": 0} | kw
    return fa.cache._APPEND.pack(*(x for v in f.values() for x in (v if isinstance(v, list) else [v])))


def _cached(**kw):
    f = CACHE | {"q": 16, "o": 16, "strides": [64] * 3, "heads": 4, "window": 0, "sinks": 0, "scale": 0.1, "dtype": 0} | kw
    return fa.cache._CACHED.pack(*(x for v in f.values() for x in (v if isinstance(v, list) else [v])))


@pytest.mark.parametrize("change,match", [
    ({"batch": 0}, "must be positive"), ({"tokens": 0}, "must be positive"), ({"heads": 5}, "multiple of kv_heads"),
    ({"d": 80}, "head_dim"), ({"page": 12}, "power of two"), ({"page": 512}, "power of two"), ({"pages": 0}, "must be positive"),
    ({"most": 0}, "must be positive"), ({"ts": 2}, "max_pages"), ({"most": 1 << 28, "ts": 1 << 28}, "2\\^31"), ({"dtype": 2}, "dtype"),
    ({"cdtype": 1}, "tensors' type"), ({"ks": 0}, "scales"), ({"cdtype": 0}, "16-bit one has none"), ({"k": 8}, "16-byte aligned"),
    ({"k0": 4104}, "multiples of 16"), ({"table": 0}, "must be given"), ({"lengths": 0}, "must be given"), ({"strides": [4] * 9}, "multiples of 8"),
])
def test_cache_refusals(change, match):
    import re

    rc, message = _call("fa_append_kv", _append(**change), None)
    assert rc == _C.FA_ERR_INVALID_ARGUMENT and re.search(match, message), message
    change = {k: v[:3] if isinstance(v, list) else v for k, v in change.items()}
    for entry, rest in (("fa_cached_attention", (None, 0, None)), ("fa_cached_workspace_size", (None,))):
        rc, message = _call(entry, _cached(**change), *rest)
        assert rc == _C.FA_ERR_INVALID_ARGUMENT and re.search(match, message), message


@pytest.mark.parametrize("change,match", [
    ({"cos": 0}, "go together"), ({"rotary": 24}, "rotary_dim"), ({"rotary": 80}, "rotary_dim"), ({"rows": 0}, "rotary_dim"),
    ({"qo": 0}, "must be present"), ({"kn": 0}, "must be present"),
])
def test_append_refusals(change, match):
    rc, message = _call("fa_append_kv", _append(**change), None)
    assert rc == _C.FA_ERR_INVALID_ARGUMENT and match in message, message


def test_python_checks_come_before_the_library():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.forward_window(q, q, q, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.window_attention(q, q, q, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.PagedKVCache(q, q)


def test_oracle_gradient_against_differences():
    gen = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((1, 4, 9, 8), (1, 2, 12, 8), (1, 2, 12, 8), (1, 4, 9, 8)))
    grads = oracle.window_backward(do, q, k, v, 4, 2)[:3]
    for i in range(3):
        args = [q, k, v]
        step = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        value = lambda h: (oracle.window_forward(*args[:i], args[i] + h * step, *args[i + 1:], 4, 2)[0] * do).sum()  # noqa: E731
        h = 1e-5  # truncation h^2 and cancellation 1e-16 / h, both below 1e-8 of the value
        assert abs((value(h) - value(-h)) / (2 * h) - (grads[i] * step).sum()) < 1e-7


def test_block_scale_of_the_oracle():
    for amax, want in ((0.0, 2.0**-60), (448.0, 1.0), (448.5, 2.0), (1.0, 2.0**-8), (1.75, 2.0**-8), (1.76, 2.0**-7), (1e-30, 2.0**-60)):
        assert oracle.power_of_two(amax) == want
