"""CPU checks of the entry points of drafted tokens: exports, refusals before
any HIP call, kernels and workspaces of a shape."""
import ctypes
import os
import re
import subprocess

import pytest

from tests.test_attention_api import GEOM, NULL, OK, TYPE, dry, ptr

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F = ctypes.c_void_p(0x10000)


@pytest.fixture(scope="module")
def lib():
    from inferflux_amd import _lib
    return _lib.load()


def test_exports_what_the_header_declares(lib):
    from inferflux_amd import _lib
    text = open(os.path.join(ROOT, "include", "ifx_drafts.h")).read()
    syms = set(re.findall(r"^\s*(?:int|int64_t)\s+(ifx_\w+)\s*\(", text, re.M))
    assert syms == {"ifx_plan_tree", "ifx_attn_tree", "ifx_attn_tree_workspace_bytes", "ifx_verify_workspace_bytes", "ifx_verify",
                    "ifx_keep_path", "ifx_plan_kept"}
    assert syms <= set(_lib.SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", _lib.LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    assert syms <= set(re.findall(r"\bT (ifx_\w+)", out))


def test_header_is_plain_c(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "ifx_drafts.h"\nint main(void) { return IFX_KEPT_NO_SPACE - 1; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-c", "-I" + os.path.join(ROOT, "include"),
                    str(src), "-o", str(tmp_path / "t.o")], check=True)


TREE = dict(parents=ptr(0), cu=ptr(1), kv=ptr(2), B=4, T=32, pos=ptr(3), masks=ptr(4), stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, OK), (dict(T=0, parents=None, pos=None, masks=None), OK), (dict(B=0), GEOM), (dict(B=4097), GEOM),
    (dict(T=-1), GEOM), (dict(T=1 << 30), GEOM), (dict(parents=None), NULL), (dict(cu=None), NULL),
    (dict(kv=None), NULL), (dict(pos=None), NULL), (dict(masks=None), NULL), (dict(pos=ptr(0)), GEOM),
    (dict(masks=ptr(2)), GEOM), (dict(masks=ptr(3)), GEOM)])
def test_plan_tree_refusals(lib, change, want):
    with dry(lib) as d:
        assert lib.ifx_plan_tree(*{**TREE, **change}.values()) == want
    assert d.text == ("k_plan_tree" if want == OK and change.get("T") != 0 else "")


ATTN = dict(q=F, qs=2048, dt=1, kc=F, vc=F, pages=100, page=64, table=F, width=50, cu=F, kv=F, masks=F, B=4,
            T=24, Hq=16, Hkv=2, D=128, max_q=4, max_kv=3000, scale=0.1, out=F, os=2048, odt=1, ws=F,
            wn=64 << 20, stream=None)


@pytest.mark.parametrize("change,want", [
    # up to 32 rows of 16 units, 24 of 64, 16 of more; blocks of 32 rows: 112 of all units
    ({}, "k_attn_rows<1,128,1>"), (dict(dt=2), "k_attn_rows<2,128,1>"), (dict(max_q=3, B=32), "k_attn_rows<1,128,1>"),
    (dict(max_q=4, B=9), "k_attn_tile<1,128,1,1>"), (dict(max_q=2, B=33), "k_attn_rows<1,128,1>"),
    (dict(max_q=3, B=33), "k_attn_tile<1,128,1,1>"), (dict(max_q=56, B=4), "k_attn_rows<1,128,1>"),
    (dict(max_q=57, B=4), "k_attn_tile<1,128,1,1>"), (dict(dt=2, max_q=57, B=4), "k_attn_tile<2,128,1,1>"),
    (dict(max_q=64), "k_attn_tile<1,128,1,1>"), (dict(max_q=65), GEOM), (dict(max_q=0), GEOM),
    (dict(masks=None), NULL), (dict(T=0, masks=None), OK), (dict(dt=0), TYPE), (dict(odt=3), TYPE),
    (dict(page=24), GEOM), (dict(D=80), GEOM), (dict(Hq=15), GEOM), (dict(scale=0.0), GEOM),
    (dict(ws=None), NULL), (dict(wn=1000), GEOM), (dict(kv=None), NULL), (dict(qs=100), GEOM)])
def test_attn_tree_kernels_and_refusals(lib, change, want):
    with dry(lib) as d:
        rc = lib.ifx_attn_tree(*{**ATTN, **change}.values())
    assert (d.text, rc) == (want, OK) if isinstance(want, str) else (rc, d.text) == (want, "")


@pytest.mark.parametrize("B,T,Hq,Hkv,D,max_q,max_kv", [
    (1, 1, 16, 2, 128, 1, 3000), (4, 24, 16, 2, 128, 6, 3000), (16, 96, 40, 8, 128, 6, 9000), (1, 61, 16, 2, 128, 61, 3000),
    (4096, 4096, 8, 8, 256, 64, 1 << 20), (1, 64, 64, 1, 256, 64, 1 << 30)])
def test_attn_tree_workspace(lib, B, T, Hq, Hkv, D, max_q, max_kv):
    """As many bytes as it says are enough, one less is not."""
    n = lib.ifx_attn_tree_workspace_bytes(B, T, Hq, Hkv, D, max_q, max_kv)
    assert 0 < n <= 64 << 20
    change = dict(B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, max_q=max_q, max_kv=max_kv, qs=Hq * D, os=Hq * D)
    for have, want in ((n, OK), (n - 1, GEOM)):
        with dry(lib) as d:
            assert lib.ifx_attn_tree(*{**ATTN, **change, "wn": have}.values()) == want
        assert d.text.startswith("k_attn_") == (want == OK)


VERIFY = dict(tokens=ptr(0), parents=ptr(1), cu=ptr(2), B=4, T=32, max_q=8, p=ptr(3), ps=1000, q=None, qs=0,
              dt=0, V=1000, au=ptr(4), su=ptr(5), acc=ptr(6), path=ptr(7), out=ptr(8), ws=ptr(16),
              wn=64 << 20, stream=None)
CHAIN = dict(parents=None, q=ptr(9), qs=1000)


@pytest.mark.parametrize("change,want", [
    ({}, OK), (CHAIN, OK), (dict(parents=None), OK), (dict(dt=1), OK), (dict(dt=2), OK), (dict(dt=3), TYPE),
    (dict(B=0), GEOM), (dict(B=4097), GEOM), (dict(T=-1), GEOM), (dict(max_q=0), GEOM), (dict(max_q=65), GEOM),
    (dict(V=0), GEOM), (dict(V=(1 << 30) + 1, ps=1 << 31), GEOM), (dict(ps=999), GEOM),
    (dict(q=ptr(9), qs=1000), GEOM), ({**CHAIN, "qs": 999}, GEOM), (dict(tokens=None), NULL), (dict(cu=None), NULL),
    (dict(p=None), NULL), (dict(au=None), NULL), (dict(su=None), NULL), (dict(acc=None), NULL),
    (dict(path=None), NULL), (dict(out=None), NULL), (dict(ws=None), NULL), (dict(wn=32768), GEOM),
    (dict(ws=ctypes.c_void_p(0x10080)), GEOM), (dict(path=ptr(0)), GEOM), (dict(out=ptr(7)), GEOM),
    (dict(acc=ptr(5)), GEOM), (dict(T=0, tokens=None, p=None, au=None, path=None, out=None), OK)])
def test_verify_refusals(lib, change, want):
    args = {**VERIFY, **change}
    with dry(lib) as d:
        assert lib.ifx_verify(*args.values()) == want
    assert d.text == (f"k_verify<{args['dt']}>" if want == OK else "")


@pytest.mark.parametrize("B,V", [(1, 1), (1, 1 << 30), (4096, 1 << 30), (32, 151936), (1, 151936), (4096, 1)])
def test_verify_workspace(lib, B, V):
    n = lib.ifx_verify_workspace_bytes(B, V)
    assert 32768 + 16 * B <= n <= 64 << 20


def test_verify_workspace_of_no_shape(lib):
    assert lib.ifx_verify_workspace_bytes(0, 5) == lib.ifx_verify_workspace_bytes(1, 0) == 0


KEEP = dict(k=F, v=F, s=None, eb=2, pages=100, page=64, Hkv=2, D=128, table=F, width=50, cu=F, kv=F, path=F,
            acc=F, B=4, T=32, max_q=8, stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, "k_keep_path<8>"), (dict(eb=1, s=F), "k_keep_path<16>"), (dict(eb=1), NULL), (dict(eb=4), TYPE),
    (dict(T=0, k=None), OK), (dict(page=8), GEOM), (dict(pages=0), GEOM), (dict(pages=1 << 26), GEOM),
    (dict(Hkv=0), GEOM), (dict(D=260), GEOM), (dict(D=100), GEOM), (dict(eb=1, s=F, D=72), GEOM),
    (dict(width=0), GEOM), (dict(width=1 << 25), GEOM), (dict(B=0), GEOM), (dict(max_q=65), GEOM),
    (dict(max_q=0), GEOM), (dict(path=None), NULL), (dict(acc=None), NULL), (dict(table=None), NULL),
    (dict(v=None), NULL), (dict(k=ctypes.c_void_p(0x10008)), GEOM)])
def test_keep_refusals(lib, change, want):
    with dry(lib) as d:
        rc = lib.ifx_keep_path(*{**KEEP, **change}.values())
    assert (d.text, rc) == (want, OK) if isinstance(want, str) else (rc, d.text) == (want, "")


KEPT = dict(cu=ptr(0), kv=ptr(1), acc=ptr(2), table=ptr(3), width=8, free=ptr(4), cap=16, count=ptr(5), page=64,
            B=4, ctx=ptr(6), left=ptr(7), status=ptr(8), stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, OK), (dict(cap=0, free=None), OK), (dict(free=None), NULL), (dict(cap=-1), GEOM), (dict(page=24), GEOM),
    (dict(B=0), GEOM), (dict(B=4097), GEOM), (dict(width=0), GEOM), (dict(acc=None), NULL), (dict(kv=None), NULL),
    (dict(count=None), NULL), (dict(ctx=None), NULL), (dict(status=None), NULL), (dict(left=ptr(5)), GEOM),
    (dict(ctx=ptr(1)), GEOM), (dict(status=ptr(7)), GEOM)])
def test_plan_kept_refusals(lib, change, want):
    with dry(lib) as d:
        assert lib.ifx_plan_kept(*{**KEPT, **change}.values()) == want
    assert d.text == ("k_plan_kept" if want == OK else "")


def test_python_refusals():
    import torch
    from inferflux_amd import drafts
    x = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        drafts.plan_tree(x, x, x)  # on the host
    with pytest.raises(ValueError):
        drafts.verify(x, x, torch.zeros(4, 8), torch.zeros(4), torch.zeros(3), 4)
