"""CPU checks of the attention entry points: exports, refusals before any HIP
call, the kernel and the split that a shape gets, workspace sizes."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F = ctypes.c_void_p(0x10000)
OK, TYPE, GEOM, NULL = 0, 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    from inferflux_amd import _lib
    return _lib.load()


def test_exports_what_the_header_declares(lib):
    from inferflux_amd import _lib
    text = open(os.path.join(ROOT, "include", "ifx_attention.h")).read()
    syms = set(re.findall(r"^\s*(?:int|int64_t)\s+(ifx_\w+)\s*\(", text, re.M))
    assert syms == {"ifx_plan_batch", "ifx_rope_append", "ifx_attn_paged_workspace_bytes",
                    "ifx_attn_paged", "ifx_attn_prompt"}
    assert syms <= set(_lib.SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", _lib.LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    assert syms <= set(re.findall(r"\bT (ifx_\w+)", out))


def test_header_is_plain_c(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "ifx_attention.h"\nint main(void) { return IFX_PLAN_NO_PAGES - 1; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-c", "-I" + os.path.join(ROOT, "include"),
                    str(src), "-o", str(tmp_path / "t.o")], check=True)


class dry:
    def __init__(self, lib):
        self.lib = lib

    def __enter__(self):
        self.lib.ifx_launch_log_begin(1)
        return self

    def __exit__(self, *e):
        self.text = self.lib.ifx_launch_log_end().decode()
        return False


def ptr(i):
    return ctypes.c_void_p(0x10000 + 0x1000 * i)


PLAN = dict(ctx=ptr(0), new=ptr(1), table=ptr(2), width=8, free=ptr(3), cap=16, count=ptr(4), page=64,
            B=4, T=32, cu=ptr(5), kv=ptr(6), pos=ptr(7), slots=ptr(8), left=ptr(9), status=ptr(10),
            stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, OK), (dict(page=24), GEOM), (dict(page=8), GEOM), (dict(page=512), GEOM), (dict(B=0), GEOM),
    (dict(B=4097), GEOM), (dict(width=0), GEOM), (dict(cap=-1), GEOM), (dict(T=-1), GEOM),
    (dict(ctx=None), NULL), (dict(table=None), NULL), (dict(status=None), NULL), (dict(pos=None), NULL),
    (dict(T=0, pos=None, slots=None), OK), (dict(cap=0, free=None), OK), (dict(free=None), NULL),
    (dict(left=ptr(4)), GEOM), (dict(kv=ptr(0)), GEOM), (dict(slots=ptr(3)), GEOM)])
def test_plan_refusals(lib, change, want):
    with dry(lib) as d:
        assert lib.ifx_plan_batch(*{**PLAN, **change}.values()) == want
    assert d.text == ("k_plan_batch" if want == OK else "")


APPEND = dict(q=F, qs=2048, k=F, ks=256, v=F, vs=256, src=0, pos=F, slots=F, freq=F, rot=128, inter=0,
              T=4, Hq=16, Hkv=2, D=128, qo=F, qos=2048, kc=F, vc=F, dt=1, pages=10, page=64, stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, OK), (dict(T=0, q=None), OK), (dict(T=-1), GEOM), (dict(src=3), TYPE), (dict(dt=0), TYPE),
    (dict(page=48), GEOM), (dict(pages=0), GEOM), (dict(pages=1 << 26), GEOM), (dict(D=132), GEOM),
    (dict(D=264), GEOM), (dict(rot=8), GEOM), (dict(rot=144), GEOM), (dict(qs=2047), GEOM),
    (dict(ks=255), GEOM), (dict(vs=0), GEOM), (dict(qos=100), GEOM), (dict(Hkv=0), GEOM),
    (dict(q=None), NULL), (dict(slots=None), NULL), (dict(freq=None), NULL), (dict(pos=None), NULL),
    (dict(freq=None, pos=None, rot=0), OK), (dict(kc=ctypes.c_void_p(0x10008)), GEOM)])
def test_append_refusals(lib, change, want):
    with dry(lib):
        assert lib.ifx_rope_append(*{**APPEND, **change}.values()) == want


PAGED = dict(q=F, qs=2048, dt=1, kc=F, vc=F, pages=100, page=64, table=F, width=20, cu=F, kv=F, B=4, T=4,
             Hq=16, Hkv=2, D=128, max_q=1, max_kv=1000, scale=0.1, window=0, out=F, os=2048, odt=1,
             ws=F, wsn=64 << 20, stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, OK), (dict(T=0, q=None), OK), (dict(dt=0), TYPE), (dict(odt=3), TYPE), (dict(page=24), GEOM),
    (dict(pages=0), GEOM), (dict(width=0), GEOM), (dict(width=1 << 26), GEOM), (dict(B=0), GEOM),
    (dict(B=4097), GEOM), (dict(Hq=15), GEOM), (dict(Hkv=0), GEOM), (dict(D=80), GEOM),
    (dict(max_q=0), GEOM), (dict(max_kv=0), GEOM), (dict(scale=0.0), GEOM), (dict(scale=-1.0), GEOM),
    (dict(scale=float("nan")), GEOM), (dict(scale=float("inf")), GEOM), (dict(window=-1), GEOM),
    (dict(qs=2047), GEOM), (dict(os=2047), GEOM), (dict(q=None), NULL), (dict(kv=None), NULL),
    (dict(ws=None, wsn=0), NULL), (dict(wsn=4096), GEOM), (dict(ws=ctypes.c_void_p(0x10010)), GEOM),
    (dict(vc=ctypes.c_void_p(0x10002)), GEOM), (dict(T=1 << 28), GEOM),
    (dict(Hq=1 << 15, Hkv=1 << 15, qs=1 << 22, os=1 << 22, T=4), GEOM)])
def test_paged_refusals(lib, change, want):
    with dry(lib) as d:
        assert lib.ifx_attn_paged(*{**PAGED, **change}.values()) == want
    assert bool(d.text) == (want == OK and change.get("T") != 0)


PROMPT = dict(q=F, qs=2048, k=F, ks=256, v=F, vs=256, dt=2, cu=F, B=3, T=100, Hq=16, Hkv=2, D=128,
              max_len=60, causal=1, window=0, scale=0.1, out=F, os=2048, odt=0, stream=None)


@pytest.mark.parametrize("change,want", [
    ({}, OK), (dict(T=0, q=None), OK), (dict(dt=0), TYPE), (dict(odt=4), TYPE), (dict(D=32), GEOM),
    (dict(max_len=0), GEOM), (dict(causal=0), OK), (dict(causal=0, window=4), GEOM),
    (dict(window=4), OK), (dict(ks=128), GEOM), (dict(vs=128), GEOM), (dict(Hq=17), GEOM),
    (dict(cu=None), NULL), (dict(v=None), NULL), (dict(B=0), GEOM)])
def test_prompt_refusals(lib, change, want):
    with dry(lib):
        assert lib.ifx_attn_prompt(*{**PROMPT, **change}.values()) == want


def test_workspace_fits_the_documented_size(lib):
    """Whatever the shape, the workspace stays within IFX_ATTN_WORKSPACE_BYTES,
    and a shape that cannot be split needs none."""
    ws = lib.ifx_attn_paged_workspace_bytes
    for B in (1, 3, 32, 300, 4096):
        for Hq, Hkv in ((1, 1), (16, 2), (40, 8), (128, 128), (256, 1)):
            for D in (64, 96, 128, 256):
                for max_q in (1, 4, 100, 4000):
                    for max_kv in (1, 100, 5000, 1 << 20):
                        n = ws(B, B * max_q, Hq, Hkv, D, max_q, max_kv)
                        assert 0 <= n <= 64 << 20
                        if max_kv <= 64:
                            assert n == 0
    assert ws(1, 1, 16, 2, 128, 1, 3000) > 0
    assert ws(0, 1, 16, 2, 128, 1, 3000) == 0


def test_wrapper_refusals_without_a_gpu():
    """Shapes and types the Python wrappers refuse before they touch a stream."""
    import torch
    from inferflux_amd import attention as at
    with pytest.raises(ValueError):
        at.kv_cache(4, 2, 128, page_size=24, device="cpu")
    with pytest.raises(ValueError):
        at.kv_cache(4, 2, 128, dtype=torch.float32, device="cpu")
    k, v = at.kv_cache(4, 2, 128, page_size=16, device="cpu")
    assert k.shape == (4, 2, 16, 16, 8) and v.shape == (4, 2, 2, 128, 8)
    i = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(1, 4, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensor"):
        at.paged_attention(q, k, v, i[:1, None], i, i[:1], 1, 1)
    with pytest.raises(ValueError, match="device tensor"):
        at.rope_append(q, q[:, :2], q[:, :2], i[:1], i[:1], k, v)
    with pytest.raises(ValueError, match="device tensor"):
        at.plan_batch(i, i, i[:, None], i, i[:1], 16, 1)
    with pytest.raises(ValueError, match="device tensor"):
        at.prompt_attention(q, q[:, :2], q[:, :2], i, 1)
    with pytest.raises(ValueError, match="as kv_cache makes"):
        at._caches(k, k)
    with pytest.raises(TypeError):
        at._caches(k, v.bfloat16())
    with pytest.raises(ValueError, match="one after the other"):
        at._rows(torch.zeros(3, 2, 16)[:, :, ::2], "q", 3, 2, 8)
    with pytest.raises(ValueError, match=r"must be \[3, 2, 8\]"):
        at._rows(torch.zeros(3, 2, 16), "q", 3, 2, 8)
    assert at._rows(torch.zeros(3, 40)[:, 8:24].view(3, 2, 8), "q", 3, 2, 8)[1] == 40


def test_outputs_are_allocated_on_the_stream_of_the_call(monkeypatch):
    """An output that a call makes for a given stream comes from that stream's
    own memory, which nothing pending on another stream still uses, and the
    current stream, where the caller goes on with it, is known to use it too."""
    import contextlib

    import torch
    from inferflux_amd import attention as at
    now, log = ["current"], []

    class Out:
        def record_stream(self, s):
            log.append(("used on", s))

    @contextlib.contextmanager
    def on(s):
        now.append(s)
        yield
        now.pop()

    def empty(*a, **k):
        log.append(("made on", now[-1]))
        return Out()

    like = torch.zeros(1)
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: now[-1])
    monkeypatch.setattr(torch, "empty", empty)
    at._new((2, 3), torch.float16, like, None)
    assert log == [("made on", "current")]
    log.clear()
    at._new((2, 3), torch.float16, like, "given")
    assert log == [("made on", "given"), ("used on", "current")]


def test_loads_of_packed_rows_are_bounded_by_the_lanes_offsets(tmp_path):
    """Stages of packed rows rely on the buffer's end for the rows behind a
    prompt's last.  The range check counts a lane's offset and not the scalar
    one, so no such load may have a scalar offset."""
    from inferflux_amd import build
    out = tmp_path / "attn_tile.s"
    subprocess.run([build.HIPCC] + build.COMMON + ["-S", "--cuda-device-only", "-x", "hip",
                    os.path.join(build.CSRC, "attn_tile.hip"), "-o", str(out)], check=True,
                   capture_output=True)
    loads = re.findall(r"buffer_load_dwordx4 \S+ \S+ (\S+) offen.* lds", out.read_text())
    assert len(loads) > 64 and set(loads) == {"0"}


def test_counts_that_pass_32_bits_are_refused():
    """A window of 2^32 + 1 keys is not one of 1; sizes below 0 are refused as
    every other bad size."""
    from inferflux_amd import attention as at
    for v in (0, 5, 2 ** 31 - 1):
        assert at._count(v, "n") == v
    for v in (-1, 2 ** 31, 2 ** 32 + 1, -2 ** 32):
        with pytest.raises(ValueError, match="window"):
            at._count(v, "window")
    with pytest.raises(ValueError, match="max_kv"):
        at.paged_workspace_bytes(1, 1, 16, 2, 128, 1, 2 ** 32 + 3000)


def test_output_types_that_no_kernel_writes():
    import torch
    from inferflux_amd import attention as at
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    for dt in (torch.float64, torch.int8):
        with pytest.raises(TypeError):
            at._out(q, None, dt, None)
        with pytest.raises(TypeError):
            at._out(q, q.to(dt), None, None)
    assert at._out(q, None, torch.float32, None).dtype is torch.float32
    assert at._out(q, None, None, None).dtype is torch.float16


@pytest.mark.parametrize("T,want", [((1 << 30), OK), ((1 << 30) + 1, GEOM), (2 ** 31 - 1, GEOM)])
def test_plan_rows_that_fit_the_grid(lib, T, want):
    with dry(lib):
        assert lib.ifx_plan_batch(*{**PLAN, "T": T}.values()) == want


@pytest.mark.parametrize("T,want", [((1 << 27) - 8, OK), ((1 << 27) - 7, GEOM), (2 ** 31 - 1, GEOM)])
def test_append_rows_that_fit_the_grid(lib, T, want):
    """A launch has less than 2^32 threads: eight tokens a workgroup of 256."""
    with dry(lib):
        assert lib.ifx_rope_append(*{**APPEND, "T": T}.values()) == want


@pytest.mark.parametrize("scale,want", [(2.3e38, OK), (2.4e38, GEOM), (3.4e38, GEOM)])
def test_scales_that_pass_fp32_with_log2_e(lib, scale, want):
    """The kernels' factor is scale log2 e: as an infinity it makes scores of 0
    no numbers."""
    with dry(lib):
        assert lib.ifx_attn_paged(*{**PAGED, "scale": scale}.values()) == want
        assert lib.ifx_attn_prompt(*{**PROMPT, "scale": scale}.values()) == want
