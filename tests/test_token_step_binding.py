"""The token-step calls of Python with the extension module and without it (no GPU needed but for the last)."""
import os
import subprocess
import sys

import pytest

import tadma_b200 as tb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def planned(python):
    """The commands of a build from nothing with that Python."""
    r = subprocess.run(["make", "-s", "-n", "-B", "-C", os.path.join(ROOT, "tadma_b200", "csrc"), f"PYTHON={python}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_library_is_built_without_python_headers(tmp_path):
    other = tmp_path / "python"  # one that says where its headers would be, but has none
    other.write_text(f'#!/bin/sh\n{sys.executable} "$@" | sed "s,^/.*,{tmp_path}/include,"\n')
    other.chmod(0o755)
    for python in (str(other), "false"):
        plan = planned(python)
        assert "libtadma_b200.so" in plan and "pycall.c" not in plan


def test_module_is_named_for_its_python():
    import sysconfig
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        pytest.skip("no headers of this Python")
    assert "_pycall" + sysconfig.get_config_var("EXT_SUFFIX") in planned(sys.executable)


@pytest.fixture(params=["module", "ctypes"])
def calls(request, monkeypatch):
    tb._load_steps()
    if request.param == "ctypes":
        monkeypatch.setattr(tb, "_calls", tb._CtypesCalls())
    return request.param


def test_a_missing_module_leaves_ctypes(monkeypatch):
    monkeypatch.setitem(sys.modules, "tadma_b200._pycall", None)  # an import of it fails
    monkeypatch.delattr(tb, "_pycall", raising=False)
    monkeypatch.setattr(tb, "_calls", None)
    assert isinstance(tb._load_steps(), tb._CtypesCalls)


def test_refusals_are_the_same(calls):
    import torch
    x, codes, scales, out = torch.zeros(2, 64).half(), torch.zeros(5, 32).byte(), torch.zeros(5, 2).half(), torch.zeros(2, 5).half()
    for text, args in (("must be \\[m, n\\]", (x, codes, scales, out.t())), ("x must be float16", (x.float(), codes, scales, out)),
                       ("unknown dtype", (x, codes, scales.to(torch.complex64), out)),
                       ("rank out of range", (x.reshape([1] * 8 + [2, 64]), codes, scales, out)), ("scales is NULL", (x, codes, None, out))):
        with pytest.raises(tb.TadmaError, match=text):
            tb.matvec_q4(*args, stream=0)
    with pytest.raises(TypeError, match="descriptor"):
        tb.matvec_q4(b"not one", codes, scales, out, stream=0)
    i = [torch.zeros(n, dtype=torch.int32) for n in (3, 3, 50, 1, 9, 4, 3, 1)]
    with pytest.raises(tb.TadmaError, match="page_size"):
        tb.block_tables(*i[:4], 1 << 40, torch.zeros((3, 8), dtype=torch.int32), *i[4:], stream=0)
    rows = torch.zeros(2, 3, 64).half()
    cache = (torch.zeros(4, 2, 16, 32).byte(), torch.zeros(4, 2, 16, 1, 2).half())
    with pytest.raises(tb.TadmaError, match="k must be"):
        tb.kv4_append(rows, rows, torch.zeros(2, dtype=torch.int64), *cache, *cache, stream=0)
    with pytest.raises(tb.TadmaError, match="k_out must be"):
        tb.kv4_read(*cache, *cache, torch.zeros(2, dtype=torch.int64), rows, rows, stream=0)
    with pytest.raises(tb.TadmaError, match="kv_heads must divide"):
        tb.kv4_attention(rows, *cache, *cache, torch.zeros((2, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 0.125, rows, stream=0)
    with pytest.raises(tb.TadmaError, match="ids come with"):
        tb.adjust_logits(out, torch.zeros((2, 1), dtype=torch.int32), None, None, out, stream=0)


@pytest.mark.gpu
def test_steps_are_the_same(calls):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(3)
    requests, heads, kv_heads, dim, page = 40, 8, 2, 64, 16
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731

    def step():
        table, slots = torch.full((requests, 60), -1, dtype=torch.int32, device="cuda"), torch.empty(requests * 200, dtype=torch.int64, device="cuda")
        starts, lens, left = ints([0] * (requests + 1)), ints([0] * requests), ints([0])
        tb.block_tables(ints([0] * requests), ints([200] * requests), torch.arange(600, dtype=torch.int32, device="cuda"), ints([600]), page, table,
                        slots, starts, lens, left)
        caches = [(torch.zeros((600, kv_heads, page, dim // 2), dtype=torch.uint8, device="cuda"),
                   torch.zeros((600, kv_heads, page, 2, 2), dtype=torch.float16, device="cuda")) for _ in range(2)]
        k, v = (torch.randn((requests * 200, kv_heads, dim), device="cuda", generator=gen).half() for _ in range(2))
        tb.kv4_append(k, v, slots, *caches[0], *caches[1])
        back = [torch.empty_like(k) for _ in range(2)]
        tb.kv4_read(*caches[0], *caches[1], slots, *back)
        q = torch.randn((requests, heads, dim), device="cuda", generator=gen).half()
        out = torch.empty_like(q)
        tb.kv4_attention(q, *caches[0], *caches[1], table, lens, 0.125, out)
        codes = torch.randint(0, 256, (100, heads * dim // 2), dtype=torch.uint8, device="cuda", generator=gen)
        y = torch.empty((requests, 100), device="cuda")
        tb.matvec_q4(out.view(requests, -1), codes, torch.full((100, 4), 0.1, device="cuda"), y)
        z = torch.empty_like(y)
        tb.adjust_logits(y, ints([[3]] * requests), ints([0] * requests), ints([1] * requests), z, presence=torch.ones(requests, device="cuda"))
        return [table, slots, starts, lens, left, *back, out, y, z]

    got = step()
    assert tb.error_flags() == 0
    tb._calls = tb._load_steps()
    gen.manual_seed(3)
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
