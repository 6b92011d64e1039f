"""The attention operators without a GPU: refusals of the C ABI and of the
Python calls, rotary tables, the cache's tensors."""
import ctypes
import math

import pytest
import torch

P = 1 << 20  # a 16-byte aligned address that is never used


def lib():
    from qwen_wlqfastshot_helen_beta_b200._lib import lib
    return lib


def rope(T=1, rows=8, pages=4, Hq=4, Hkv=2, D=64, rot=64, page=16, dtype=1, ke=None, ve=None, q=P, cs=P, tok=256):
    return lib().wlq_rope_kv_write(q, P, P, P, cs, P, P, P, ke, ve, P, None, tok, 64, 128, 64, 128, 64, 256, 64, 0, 0, T,
                                   rows, pages, Hq, Hkv, D, rot, page, 0, dtype, None)


def prompt(T=2, B=1, Hq=4, Hkv=2, D=64, scale=0.1, dtype=1, tok=256, out=P):
    return lib().wlq_prompt_attention(P, P, P, P, out, tok, 64, 128, 64, 128, 64, 256, 64, T, B, Hq, Hkv, D, scale, 1,
                                      dtype, None)


def paged(T=2, B=2, Hq=4, Hkv=2, D=64, page=16, max_q=1, scale=0.1, ke=None, ve=None, cu=None, cols=4):
    return lib().wlq_paged_attention(P, P, P, ke, ve, P, P, cu, P, 256, 64, 256, 64, T, B, Hq, Hkv, D, page, 8, cols,
                                     max_q, scale, 1, None, 0, None)


def read(T=1, B=1, Hkv=2, D=64, page=16, ke=None, ve=None, out=P):
    return lib().wlq_kv_read(P, P, ke, ve, P, P, out, P, T, B, 8, 4, Hkv, D, page, 1, None)


@pytest.mark.parametrize("call,code,word", [
    (lambda: rope(T=-1), 1, b"T=-1"), (lambda: rope(rows=0), 1, b"table rows"), (lambda: rope(dtype=5), 2, b"act_dtype"),
    (lambda: rope(Hq=5), 1, b"heads"), (lambda: rope(D=72), 2, b"head size"), (lambda: rope(D=512), 2, b"head size"),
    (lambda: rope(rot=40), 2, b"rotated"), (lambda: rope(rot=80), 2, b"rotated"), (lambda: rope(page=8), 2, b"page_size"),
    (lambda: rope(page=48), 2, b"page_size"), (lambda: rope(ke=P), 1, b"k_exp"), (lambda: rope(q=P + 8), 3, b"aligned"),
    (lambda: rope(tok=250), 3, b"aligned"), (lambda: rope(cs=P + 4), 3, b"cos_sin"), (lambda: rope(cs=None), 1, b"cos_sin"),
    (lambda: prompt(D=80), 2, b"head size"), (lambda: prompt(scale=0.0), 1, b"scale"),
    (lambda: prompt(scale=float("nan")), 1, b"scale"), (lambda: prompt(scale=float("inf")), 1, b"scale"),
    (lambda: prompt(Hq=6, Hkv=4), 1, b"heads"), (lambda: prompt(Hq=129, Hkv=1), 2, b"128 query heads"),
    (lambda: prompt(out=None), 1, b"out"), (lambda: prompt(out=P + 2), 3, b"aligned"), (lambda: prompt(B=0), 1, b"cu_seqlens"),
    (lambda: paged(D=96), 2, b"head size"), (lambda: paged(T=3), 1, b"without cu_q"), (lambda: paged(max_q=2), 1, b"without cu_q"),
    (lambda: paged(max_q=0), 1, b"size"), (lambda: paged(ke=P), 1, b"k_exp"), (lambda: paged(ke=P + 4, ve=P), 3, b"k_exp"),
    (lambda: paged(T=70000, B=70000), 2, b"sequences"), (lambda: paged(cols=1 << 30), 2, b"too many"),
    (lambda: read(D=20), 2, b"head size"), (lambda: read(out=None), 1, b"required"), (lambda: read(out=P + 4), 3, b"aligned"),
    (lambda: read(ve=P), 1, b"k_exp"),
])
def test_refusals(call, code, word):
    assert call() == code and word in lib().wlq_last_error()


def test_paged_refuses_tokens_of_no_sequence():
    """As the prompt form does: the launch would have no CTA."""
    for max_q in (1, 60):
        assert paged(T=2, B=0, cu=P, max_q=max_q) == 1 and b"sequences" in lib().wlq_last_error()


def test_paged_refuses_more_key_tiles_than_it_can_count():
    """The few-row kernel's list of tiles (64 keys of a kv head) is counted in 31 bits."""
    assert paged(T=32768, B=32768, page=128, cols=1 << 17) == 2 and b"too many" in lib().wlq_last_error()  # 2^34 tiles
    assert paged(T=32768, B=32768, page=128, cols=1 << 14) == 2 and b"too many" in lib().wlq_last_error()  # 2^31
    paged(T=32768, B=32768, page=128, cols=(1 << 14) - 1)
    assert b"too many" not in lib().wlq_last_error()


def test_nothing_to_do_is_no_error():
    assert rope(T=0) == 0 and prompt(T=0, B=0) == 0 and paged(T=0, B=0) == 0 and read(T=0, B=0) == 0


def test_python_refuses_cpu_tensors_and_wrong_arguments():
    from qwen_wlqfastshot_helen_beta_b200 import _C, _calls
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="wlq: prompt_attention: q must be a CUDA tensor"):
        _C.prompt_attention(x, x, x, i, x)
    with pytest.raises(RuntimeError, match="wlq: paged_attention: q must be a tensor"):
        _C.paged_attention(None, x, x, i, i, x)
    with pytest.raises(RuntimeError, match="wlq: kv_read: k_out must be a CUDA tensor"):
        _C.kv_read(x, x, i, i, x, x)
    with pytest.raises(RuntimeError, match="wlq: rope_kv_write: q must be a CUDA tensor"):
        _C.rope_kv_write(x, x, x, i, x, i, x, x, x)
    with pytest.raises(TypeError):
        _calls.kv_read(x)
    with pytest.raises(TypeError):
        _calls.setup((1, 2), RuntimeError)


def test_linears_do_without_the_extension_module():
    import subprocess
    import sys
    code = """
import sys
sys.modules["qwen_wlqfastshot_helen_beta_b200._calls"] = None  # as if it were not there
import numpy as np, torch
import qwen_wlqfastshot_helen_beta_b200 as pkg
from qwen_wlqfastshot_helen_beta_b200 import _C
assert hasattr(torch.ops.wlq_fastShot, "gemv") and _C.lib.wlq_abi_version() == 1
x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
try:
    _C.prompt_attention(x, x, x, x, x)
except RuntimeError as e:
    assert "wlq: prompt_attention" in str(e) and "_calls" in str(e) and "build.py" in str(e), e
    print("ok")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr


def test_attention_ops_beside_somebody_elses_linears():
    """Another plugin's wlq_fastShot::gemv leaves the attention ops where they are; a second import changes nothing."""
    import os
    import subprocess
    import sys
    code = """
import torch
lib = torch.library.Library("wlq_fastShot", "FRAGMENT")
lib.define("gemv(Tensor x) -> Tensor")
import qwen_wlqfastshot_helen_beta_b200 as pkg
for name in ("rope_kv_write", "kv_read", "prompt_attention", "paged_attention"):
    assert hasattr(torch.ops.wlq_fastShot, name), name
import gc, importlib
importlib.reload(pkg)
gc.collect()
x = torch.zeros(2, 4, 64)
try:
    torch.ops.wlq_fastShot.rope_kv_write(x, x, x, x, x, x, x, x, x)
except RuntimeError as e:
    assert "wlq: rope_kv_write: q must be a CUDA tensor" in str(e), e
    print("ok")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr


def test_the_library_is_linked_where_the_extension_module_does_not_compile(tmp_path, monkeypatch):
    import os
    import subprocess
    from qwen_wlqfastshot_helen_beta_b200 import build
    (tmp_path / "a.c").write_text("int wlq_a(void) { return 1; }")
    subprocess.run(["gcc", "-fPIC", "-c", str(tmp_path / "a.c"), "-o", str(tmp_path / "a.o")], check=True)

    def no_calls():
        raise RuntimeError("compile failed: no torch headers")

    monkeypatch.setattr(build, "_build_calls", no_calls)
    monkeypatch.setattr(build, "_compile", lambda src, verbose: str(tmp_path / "a.o"))
    monkeypatch.setattr(build.glob, "glob", lambda pattern: [str(tmp_path / "a.c")] if pattern.endswith(".cpp") else [])
    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    with pytest.raises(RuntimeError, match="no torch headers"):
        build.build()
    assert os.path.exists(build.LIB)


def test_rope_table():
    from qwen_wlqfastshot_helen_beta_b200.attention import rope_frequencies, rope_table
    t = rope_table(1000, 64, 1e4, device="cpu")
    assert t.shape == (1000, 64) and t.dtype == torch.float32
    for p, i in ((0, 0), (999, 0), (999, 31), (7, 13)):
        a = p * 1e4 ** (-2 * i / 64)
        assert abs(t[p, i].item() - math.cos(a)) < 6e-8 and abs(t[p, 32 + i].item() - math.sin(a)) < 6e-8
    lin = rope_table(100, 32, 1e4, {"type": "linear", "factor": 4.0}, device="cpu")
    assert torch.equal(lin[4::4], rope_table(25, 32, 1e4, device="cpu")[1:])  # position 4 n looks like position n
    f, a = rope_frequencies(128, 1e6, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768})
    g, _ = rope_frequencies(128, 1e6)
    assert abs(a - (0.1 * math.log(4) + 1)) < 1e-12
    assert torch.equal(f[:10], g[:10]) and torch.allclose(f[-10:], g[-10:] / 4, rtol=1e-12)  # fast pairs kept, slow ones stretched
    assert (f <= g).all() and (f >= g / 4 * (1 - 1e-12)).all() and (f[1:] < f[:-1]).all()
    d, _ = rope_frequencies(64, 1e4, {"type": "dynamic", "factor": 2.0})
    h, _ = rope_frequencies(64, 1e4)
    assert d[0] == 1.0 and abs(d[-1] / h[-1] - 0.5) < 1e-9  # the slowest pair stretched by the factor
    with pytest.raises(ValueError):
        rope_frequencies(64, 1e4, {"type": "other", "factor": 2.0})


def test_rope_dynamic_scaling_goes_by_the_length():
    """Dynamic NTK: base (f L / n - (f - 1)) ** (d / (d - 2)) beyond the n trained positions, the base as it is up to there."""
    from qwen_wlqfastshot_helen_beta_b200.attention import rope_frequencies, rope_table
    s = {"type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 4096}
    plain = rope_frequencies(64, 1e4)[0]
    for length in (None, 1, 4095, 4096):
        assert torch.equal(rope_frequencies(64, 1e4, s, length)[0], plain)
    for length, stretch in ((6144, 2.0), (8192, 3.0), (32768, 15.0)):
        got = rope_frequencies(64, 1e4, s, length)[0]
        assert got[0] == 1.0
        for i in (1, 7, 31):
            want = (1e4 * stretch ** (64 / 62)) ** (-2 * i / 64)
            assert abs(got[i].item() / want - 1) < 1e-12
    assert torch.equal(rope_table(4096, 64, 1e4, s, "cpu"), rope_table(4096, 64, 1e4, device="cpu"))
    long = rope_table(8192, 64, 1e4, s, "cpu")
    a = 8191 * (1e4 * 3.0 ** (64 / 62)) ** (-62 / 64)
    assert abs(long[8191, 31].item() - math.cos(a)) < 1e-7 and abs(long[8191, 63].item() - math.sin(a)) < 1e-7
    assert torch.equal(rope_table(4096, 64, 1e4, s, "cpu", length=8192), long[:4096])
    assert torch.equal(rope_table(8192, 64, 1e4, s, "cpu", length=4096), rope_table(8192, 64, 1e4, device="cpu"))
    bare = {"type": "dynamic", "factor": 2.0}
    with pytest.raises(ValueError, match="original_max_position_embeddings"):
        rope_table(8192, 64, 1e4, bare, "cpu")
    with pytest.warns(UserWarning, match="ntk"):
        fixed = rope_frequencies(64, 1e4, bare)[0]
    assert torch.equal(fixed, rope_frequencies(64, 1e4, {"type": "ntk", "factor": 2.0}, 100)[0])


def test_rope_scaling_as_config_files_write_it():
    """Keys with null count as absent, keys that would change the angles and are not known are refused."""
    from qwen_wlqfastshot_helen_beta_b200.attention import rope_frequencies
    s = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    f, a = rope_frequencies(128, 1e6, s)
    g, b = rope_frequencies(128, 1e6, dict(s, attention_factor=None, beta_fast=None, beta_slow=None, mscale=None))
    assert torch.equal(f, g) and a == b
    assert rope_frequencies(128, 1e6, dict(s, attention_factor=1.5, mscale=1.0))[1] == 1.5
    for bad, word in ((dict(s, mscale=1.0, mscale_all_dim=1.0), "mscale"), (dict(s, truncate=False), "truncate"),
                      ({"type": "yarn", "factor": 4.0}, "original_max"), ({"type": "linear"}, "factor"),
                      ({"type": "linear", "factor": None}, "factor")):
        with pytest.raises(ValueError, match=word):
            rope_frequencies(128, 1e6, bad)


def test_cache_tensors():
    from qwen_wlqfastshot_helen_beta_b200.attention import PagedKVCache
    c = PagedKVCache(5, 2, 64, 32, 8, torch.float16, "cpu")
    k, v, ke, ve = c.tensors
    assert k.shape == v.shape == (5, 2, 32, 64) and k.dtype == torch.float8_e4m3fn and ke.shape == (5, 2, 32)
    assert c.nbytes() == 2 * 5 * 2 * 32 * 65
    c = PagedKVCache(5, 2, 64, 32, 16, torch.float16, "cpu")
    assert c.tensors[0].dtype == torch.float16 and c.tensors[2] is None and c.nbytes() == 2 * 5 * 2 * 32 * 64 * 2
    with pytest.raises(ValueError):
        PagedKVCache(5, 2, 64, 32, 4)


ONCE = r"""
#include "wlq_once.h"
#include <cstdio>
int main() {
    wlq::OncePerDevice once;
    int calls[66] = {};
    auto at = [&](int device, cudaError_t e) { return once.run(device, [&] { ++calls[device]; return e; }); };
    bool ok = at(0, cudaErrorUnknown) == cudaErrorUnknown;       // a failure is not kept ...
    ok = ok && at(0, cudaSuccess) == cudaSuccess && calls[0] == 2;  // ... and tried again
    ok = ok && at(0, cudaErrorUnknown) == cudaSuccess && calls[0] == 2;
    ok = ok && at(1, cudaSuccess) == cudaSuccess && calls[1] == 1;  // another device has a setting of its own
    ok = ok && at(63, cudaSuccess) == cudaSuccess && at(63, cudaSuccess) == cudaSuccess && calls[63] == 1;
    ok = ok && at(64, cudaSuccess) == cudaSuccess && at(64, cudaSuccess) == cudaSuccess && calls[64] == 2;  // not remembered
    puts(ok ? "ok" : "wrong");
}
"""


def test_settings_are_made_on_every_device(tmp_path):
    import glob
    import os
    import re
    import subprocess
    from qwen_wlqfastshot_helen_beta_b200.build import CSRC, CUDA_HOME
    (tmp_path / "once.cpp").write_text(ONCE)
    exe = str(tmp_path / "once")
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, "-I", os.path.join(CUDA_HOME, "include"), str(tmp_path / "once.cpp"),
                    "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True, check=True).stdout == "ok\n"
    # no kernel's attribute is kept for the whole process
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        assert not re.search(r"static\s+(const\s+)?cudaError_t", open(path).read()), path


def test_header_constants():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = open(os.path.join(root, "include", "wlq_b200.h")).read()
    assert re.search(r"WLQ_DEVERR_POSITION 2u", src) and re.search(r"WLQ_ATTENTION_ZERO_BYTES \(256u \* 1024u\)", src)
    assert isinstance(lib().wlq_paged_attention_workspace_bytes(28, 4, 128, 1), int)
    assert ctypes.sizeof(ctypes.c_size_t) == 8
