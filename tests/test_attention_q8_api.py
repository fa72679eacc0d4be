"""CPU checks of the 8-bit cache's entry points: exports, refusals before any
HIP call, the kernel that a shape gets."""
import ctypes
import os
import re
import subprocess

import pytest

from tests.test_attention_api import GEOM, NULL, OK, TYPE, dry

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F = ctypes.c_void_p(0x10000)
ODD = ctypes.c_void_p(0x10008)


@pytest.fixture(scope="module")
def lib():
    from inferflux_amd import _lib
    return _lib.load()


def test_exports_what_the_header_declares(lib):
    from inferflux_amd import _lib
    text = open(os.path.join(ROOT, "include", "ifx_attention_q8.h")).read()
    syms = set(re.findall(r"^\s*(?:int|int64_t)\s+(ifx_\w+)\s*\(", text, re.M))
    assert syms == {"ifx_rope_append_q8", "ifx_read_rows_q8", "ifx_attn_paged_q8_workspace_bytes",
                    "ifx_attn_paged_q8"}
    assert syms <= set(_lib.SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", _lib.LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    assert syms <= set(re.findall(r"\bT (ifx_\w+)", out))


def test_header_is_plain_c(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "ifx_attention_q8.h"\nint main(void) { return 0; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-c", "-I" + os.path.join(ROOT, "include"),
                    str(src), "-o", str(tmp_path / "t.o")], check=True)


APPEND = dict(q=F, qs=2048, k=F, ks=256, v=F, vs=256, src=0, pos=F, slots=F, freq=F, rot=128, inter=0,
              T=4, Hq=16, Hkv=2, D=128, qo=F, qos=2048, qdt=1, kc=F, vc=F, s=F, pages=10, page=64, stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, OK), (dict(T=0, q=None, s=None), OK), (dict(T=-1), GEOM), (dict(src=3), TYPE), (dict(qdt=0), TYPE),
    (dict(page=48), GEOM), (dict(pages=0), GEOM), (dict(pages=1 << 26), GEOM), (dict(D=112), GEOM),
    (dict(D=288), GEOM), (dict(rot=136), GEOM), (dict(rot=144), GEOM), (dict(rot=8), GEOM),
    (dict(rot=0, pos=None, freq=None), OK), (dict(pos=None), NULL), (dict(freq=None), NULL), (dict(slots=None), NULL),
    (dict(s=None), NULL), (dict(kc=None), NULL), (dict(qo=None), NULL), (dict(ks=255), GEOM), (dict(qos=2047), GEOM),
    (dict(kc=ODD), GEOM), (dict(s=ODD), GEOM), (dict(Hq=0), GEOM), (dict(Hkv=65537), GEOM)])
def test_append_refusals(lib, change, want):
    with dry(lib) as d:
        assert lib.ifx_rope_append_q8(*{**APPEND, **change}.values()) == want
    assert d.text.startswith("k_rope_append_q8<") == (want == OK and change.get("T") != 0)


READ = dict(k=F, v=F, s=F, pages=10, page=64, slots=F, N=4, Hkv=2, D=128, ko=F, ks=256, vo=F, vs=256, dt=1,
            stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, OK), (dict(dt=0), OK), (dict(dt=2), OK), (dict(dt=3), TYPE), (dict(N=0, k=None), OK), (dict(N=-1), GEOM),
    (dict(N=1 << 27), GEOM), (dict(page=8), GEOM), (dict(pages=0), GEOM), (dict(Hkv=0), GEOM), (dict(D=48), GEOM),
    (dict(ks=255), GEOM), (dict(vs=255), GEOM), (dict(slots=None), NULL), (dict(s=None), NULL), (dict(vo=None), NULL),
    (dict(v=ODD), GEOM)])
def test_read_refusals(lib, change, want):
    with dry(lib) as d:
        assert lib.ifx_read_rows_q8(*{**READ, **change}.values()) == want
    assert d.text == (f"k_read_rows_q8<{change.get('dt', 1)}>" if want == OK and change.get("N") != 0 else "")


ATTN = dict(q=F, qs=2048, dt=1, kc=F, vc=F, s=F, pages=100, page=64, table=F, width=50, cu=F, kv=F, masks=None,
            B=4, T=24, Hq=16, Hkv=2, D=128, max_q=4, max_kv=3000, scale=0.1, window=0, out=F, os=2048, odt=1,
            ws=F, wn=64 << 20, stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, "k_attn_rows_q8<128>"), (dict(max_q=2), "k_attn_rows16_q8<128>"), (dict(dt=2), "k_attn_rows_q8<128>"),
    # blocks of 32 rows: 112 of all units, 256 where each has 8 at most
    (dict(max_q=56), "k_attn_rows_q8<128>"), (dict(max_q=57), "k_attn_tile_q8<128,1>"),
    (dict(max_q=32, B=16), "k_attn_rows_q8<128>"), (dict(max_q=33, B=16), "k_attn_tile_q8<128,1>"),
    (dict(max_q=5, B=64), "k_attn_rows_q8<128>"), (dict(max_q=5, B=65), "k_attn_tile_q8<128,1>"),
    (dict(D=64, qs=1024, os=1024), "k_attn_rows_q8<64>"), (dict(D=96), "k_attn_rows_q8<96>"),
    (dict(D=256, qs=4096, os=4096, max_q=90), "k_attn_tile_q8<256,1>"), (dict(masks=F), "k_attn_rows_q8<128>"),
    (dict(masks=F, max_q=64), "k_attn_tile_q8<128,1>"), (dict(masks=F, max_q=65), GEOM),
    (dict(max_q=256, B=1, T=256), "k_attn_tile_q8<128>"),
    (dict(masks=F, window=9), GEOM), (dict(window=9), "k_attn_rows_q8<128>"), (dict(window=-1), GEOM),
    (dict(T=0, s=None), OK), (dict(s=None), NULL), (dict(s=ODD), GEOM), (dict(kc=ODD), GEOM), (dict(dt=0), TYPE),
    (dict(odt=3), TYPE), (dict(page=24), GEOM), (dict(D=160), GEOM), (dict(Hq=15), GEOM), (dict(scale=0.0), GEOM),
    (dict(ws=None), NULL), (dict(wn=1000), GEOM), (dict(kv=None), NULL), (dict(os=100), GEOM), (dict(max_q=0), GEOM)])
def test_attention_kernels_and_refusals(lib, change, want):
    with dry(lib) as d:
        rc = lib.ifx_attn_paged_q8(*{**ATTN, **change}.values())
    assert (d.text, rc) == (want, OK) if isinstance(want, str) else (rc, d.text) == (want, "")


@pytest.mark.parametrize("B,T,Hq,Hkv,D,max_q,max_kv", [
    (1, 1, 16, 2, 128, 1, 3000), (4, 24, 16, 2, 128, 6, 3000), (16, 96, 40, 8, 128, 6, 9000), (1, 61, 16, 2, 128, 61, 3000),
    (1, 512, 40, 8, 128, 512, 8000), (4096, 4096, 8, 8, 256, 64, 1 << 20), (1, 64, 64, 1, 256, 64, 1 << 30)])
def test_attention_workspace(lib, B, T, Hq, Hkv, D, max_q, max_kv):
    """As many bytes as it says are enough, one less is not."""
    n = lib.ifx_attn_paged_q8_workspace_bytes(B, T, Hq, Hkv, D, max_q, max_kv)
    assert 0 < n <= 64 << 20
    change = dict(B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, max_q=max_q, max_kv=max_kv, qs=Hq * D, os=Hq * D)
    for have, want in ((n, OK), (n - 1, GEOM)):
        with dry(lib) as d:
            assert lib.ifx_attn_paged_q8(*{**ATTN, **change, "wn": have}.values()) == want
        assert d.text.startswith("k_attn_") == (want == OK)


def test_python_refusals():
    import torch
    from inferflux_amd import attention_q8 as q8
    for kw in (dict(page_size=24), dict(head_dim=48), dict(head_dim=512)):
        with pytest.raises(ValueError):
            q8.kv_cache(**{**dict(num_pages=2, kv_heads=2, head_dim=64, device="cpu"), **kw})
    c = q8.kv_cache(3, 2, 64, 16, device="cpu")
    x = torch.zeros(2, 2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        q8.rope_append(x, x, x, i, i, c)  # on the host
    with pytest.raises(TypeError):
        q8._q8_caches(q8.Q8Cache(c.k.half(), c.v, c.scales))
    with pytest.raises(ValueError):
        q8._q8_caches(q8.Q8Cache(c.k, c.v[:, :1], c.scales))
