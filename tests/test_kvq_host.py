"""The rotary positions and the 8-bit caches on a machine without a GPU: the argument rules, layout and key splits under
the sanitizers (tests/cpp/test_kvq_plan.cpp), the entry points' refusals that need no device, the C structs, and the
plain restatement that the GPU tests compare with (_kvq_ref.py), checked against closed forms and planted mistakes."""
from __future__ import annotations

import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

import _kvq_ref as ref
from zwhisper_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_plan_under_sanitizers(tmp_path):
    exe = str(tmp_path / "kvq_plan")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                        f"-I{ROOT}/include", f"-I{ROOT}/zwhisper_amd/csrc", os.path.join(ROOT, "tests", "cpp", "test_kvq_plan.cpp"),
                        "-o", exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-4000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "ok" in run.stdout.split(), (run.stdout + run.stderr)[-4000:]


def test_structs_match_the_header():
    """Field for field, and in zig/gpu.zig too."""
    header = open(_lib.HEADER).read()
    zig = open(os.path.join(ROOT, "zig", "gpu.zig")).read()
    for cname, zname, struct in (("zwg_rope_desc", "RopeDesc", _lib.RopeDescC), ("zwg_kvq_desc", "KvqDesc", _lib.KVQDescC),
                                 ("zwg_kvq_attn", "KvqAttn", _lib.KVQAttnC), ("zwg_kvq_cut", "KvqCut", _lib.KVQCutC)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), header, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = re.findall(r"(\w+);", body)
        want = [f for f, _ in struct._fields_]
        assert fields == want, cname
        zbody = re.search(r"pub const %s = extern struct \{(.*?)\n\};" % zname, zig, re.S).group(1)
        assert re.findall(r"^\s+([a-z_0-9]+):", zbody, re.M) == want, zname
    assert ctypes.sizeof(_lib.RopeDescC) == 3 * 8 + 8 + 2 * 8 + 8 + 3 * 8
    assert ctypes.sizeof(_lib.KVQDescC) == 6 * 8 + 8
    assert ctypes.sizeof(_lib.KVQAttnC) == 10 * 8 + 8
    assert ctypes.sizeof(_lib.KVQCutC) == 8 * 8


def test_entry_points_without_a_device():
    L = _lib.lib()
    d = _lib.KVQDescC(2, 3, 100, 2, 64, 32, 0, 0)
    units, n_pad = 12, 128
    need = 2 * units * (n_pad * 64 + n_pad // 32 * 4 + 32 * 64 * 4 + 264)
    assert need <= L.zwg_kvq_bytes(ctypes.byref(d)) <= need + 7 * 256
    d.block = 31
    assert L.zwg_kvq_bytes(ctypes.byref(d)) == 0
    assert L.zwg_kvq_bytes(None) == 0
    out = ctypes.c_void_p(5)
    for rc, msg in ((lambda: L.zwg_rope_create(None, None, ctypes.byref(out)), "null context"),
                    (lambda: L.zwg_kvq_create(None, ctypes.byref(d), None, ctypes.byref(out)), "null context"),
                    (lambda: L.zwg_rope_create(None, None, None), "null output"),
                    (lambda: L.zwg_kvq_create(None, None, None, None), "null output"),
                    (lambda: L.zwg_rope_apply_dev(None, None, 1, 1, 4, None, 0, None, 4, 0), "null rope"),
                    (lambda: L.zwg_kvq_append(None, 0, 0, 0, 1, 0, None, None, None, None, 0, 0), "null kvq"),
                    (lambda: L.zwg_kvq_append_batch(None, 0, 0, 1, None, None, None, None, None, None, 0, 0), "null kvq"),
                    (lambda: L.zwg_kvq_rows_dev(None, 0, 1, 0, 1, None, 0, 1, None, None), "null kvq"),
                    (lambda: L.zwg_kvq_attention_dev(None, 0, 0, 1, None, None, None, None), "null kvq"),
                    (lambda: L.zwg_kvq_evict_dev(None, 0, 1, 0, 1, None, None, None), "null kvq")):
        assert rc() == _lib.ZWG_ERROR
        assert msg in _lib.last_error(None)
    assert out.value is None
    L.zwg_rope_destroy(None)
    L.zwg_kvq_destroy(None)


# ---------------------------------------------------------------------------------------------- the restatement


def test_quantise_closed_forms():
    x = np.zeros((16, 32), np.float32)
    assert not ref.quantise(x, "i8").any()
    x[3, 4], x[5, 6] = 127.0, 2.5
    q = ref.quantise(x, "i8")
    assert q[3, 4] == 127.0 and q[5, 6] == 2.0  # a tie goes to even
    x[5, 6] = 3.5
    assert ref.quantise(x, "i8")[5, 6] == 4.0
    x[3, 4] = 448.0
    # steps of 2 from 16 to 32 (ties to even), of 32 above 256, subnormals in steps of 2^-9
    for a, b in ((17.0, 16.0), (19.0, 20.0), (2.0 ** -9, 2.0 ** -9), (2.0 ** -10, 0.0), (3 * 2.0 ** -10, 2.0 ** -8),
                 (-300.0, -288.0), (-304.0, -320.0), (-305.0, -320.0)):
        x[5, 6] = a
        got = float(ref.quantise(x, "e4m3")[5, 6])
        assert got == b, (a, got)
    torch = pytest.importorskip("torch")
    y = (np.random.default_rng(0).standard_normal((64, 128)) * 100).astype(np.float32)
    y[0, 0] = 448.0
    y = np.clip(y, -448, 448)
    assert np.array_equal(ref.quantise(y, "e4m3"), torch.from_numpy(y).to(torch.float8_e4m3fn).float().numpy())
    x[0, 0] = np.nan
    assert np.isnan(ref.quantise(x, "i8")).all()


def test_cache_is_of_rows_not_of_calls():
    """Whatever calls bring a block's rows, it holds what one call gives; a mistake planted in the restatement (a block
    requantised from its values) is seen."""
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((70, 2, 32)).astype(np.float32) for _ in range(2))
    whole = ref.Cache(100, 2, 32, 32, "i8")
    whole.append(0, k, v)
    for cuts in ([1] * 70, [30, 5, 35], [33, 37]):
        c, at = ref.Cache(100, 2, 32, 32, "i8"), 0
        for n in cuts:
            c.append(at, k[at: at + n], v[at: at + n])
            at += n
        assert np.array_equal(c.vals[0], whole.vals[0]) and np.array_equal(c.vals[1], whole.vals[1])
    c, at = ref.Cache(100, 2, 32, 32, "i8"), 0
    for n in [1] * 70:
        c.append(at, k[at: at + n], v[at: at + n])
        c.open = None  # the mistake
        at += n
    assert not np.array_equal(c.vals[0], whole.vals[0])


def test_attend_and_choose_closed_forms():
    rng = np.random.default_rng(2)
    v = rng.standard_normal((50, 1, 8)).astype(np.float32)
    q = np.zeros((3, 2, 8), np.float32)
    out, w, _ = ref.attend(q, v, v, 50, True)
    for i in range(3):
        assert np.allclose(out[i, 0], v[: 48 + i, 0].mean(0))
    assert np.isclose(w.sum(), 6.0) and np.isclose(w[0, 49], 2 / 50)
    assert not ref.attend(q, v, v, 2, True)[0][0].any()  # query 0 of 3 over 2 keys sees none
    assert ref.choose([1, 5, 5, 2, 5, 0], 6, 4, 0, 1) == [1, 2, 4, 5]
    assert ref.choose([1, 5, 5, 2, 5, 0], 6, 3, 1, 1) == [0, 1, 5]
    assert ref.choose([1, float("nan"), 9.0], 3, 1, 0, 0) == [1]
    assert ref.choose([3.0, 1.0], 2, 5, 1, 1) == [0, 1]


def test_rotation_closed_forms():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 2, 16)).astype(np.float32)
    for layout in ("half", "interleaved"):
        w, m = ref.rope_freqs(12, 1e4)
        y = ref.rotate(x, [0, 1, 7, 100], 12, layout, w, m)
        assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 12:], x[..., 12:])
        assert np.allclose((y ** 2).sum(-1), (x.astype(np.float64) ** 2).sum(-1), rtol=1e-6)
        back = ref.rotate(y.astype(np.float32), [0, 1, 7, 100], 12, layout, w, m, inverse=True)
        assert np.allclose(back, x, atol=1e-5)
    w1, _ = ref.rope_freqs(16, 1e4)
    w2, m2 = ref.rope_freqs(16, 1e4, "yarn", 4.0, 10 ** 9)
    assert np.allclose(w1, w2) and m2 > 1  # every pair turns often: all stay
    w2, _ = ref.rope_freqs(16, 1e4, "yarn", 4.0, 1)
    assert np.allclose(w2, w1 / 4)
    w2, _ = ref.rope_freqs(16, 1e4, "ntk", 4.0)
    assert np.isclose(w2[0], w1[0]) and np.isclose(w2[-1], w1[-1] / 4)
