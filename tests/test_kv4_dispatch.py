"""The 4-bit KV cache's entry points on the CPU: what they refuse, and what they launch
(tests/fake_hip.cpp stands in for the HIP runtime)."""
import ctypes
import json
import pathlib
import subprocess
import sys

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from csed499ii_amd import _lib  # noqa: E402
from tests.launches import _base, build_fake  # noqa: E402

NULL = ctypes.c_void_p(0)


def attention(lib, at, tokens, requests, q_heads, kv_heads, head_dim, max_q, max_kv, cu_q, groupsize=-1, stream=64):
    """One call with operands at address ``at``, which is never read on the host."""
    p = ctypes.c_void_p(at)
    return lib.marlin_hip_kv4_attention(p, p, p, p, p if cu_q else NULL, p, NULL, tokens, requests, q_heads, kv_heads,
                                        head_dim, q_heads * head_dim, head_dim, 16, 1 << 16, 1 << 14, groupsize, max_q,
                                        max_kv, 1.0, 0, 0, ctypes.c_void_p(stream))


def test_one_token_a_request_needs_as_many_tokens(built_lib):
    """Without cu_q request i is token i: fewer tokens than requests would be read past q."""
    assert attention(built_lib, 0, 3, 4, 8, 2, 128, 1, 64, False) == _lib.ERR_PROB_SHAPE
    assert "cu_q" in _lib.last_error()


@pytest.mark.parametrize("width,page,code", [(1 << 26, 16, "OK"), (1 << 22, 256, "OK"), ((1 << 26) + 1, 16, "ERR_PROB_SHAPE"),
                                             (1 << 30, 16, "ERR_PROB_SHAPE")])
def test_table_width(fake, width, page, code):
    """A table row covers 2^30 tokens at most, as attention asks for: kv_lens, cut there, is an int32."""
    assert tables_in_child(fake, width, page) == getattr(_lib, code)


@pytest.fixture(scope="module")
def fake(built_lib, tmp_path_factory):
    return build_fake(tmp_path_factory.mktemp("fake_hip"))


def launches(fake, calls):
    """Per call (the arguments of ``attention`` after ``at``) its launches: kernel, grid, and whether
    the call asked for scratch (each on a stream of its own), seen in another process."""
    out = subprocess.run([sys.executable, str(pathlib.Path(__file__)), json.dumps({"fake": str(fake), "calls": calls})],
                         capture_output=True, text=True, cwd=ROOT, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    return json.loads(out.stdout.splitlines()[-1])


def tables_in_child(fake, width, page):
    out = subprocess.run([sys.executable, str(pathlib.Path(__file__)), json.dumps({"fake": str(fake), "tables": [width, page]})],
                         capture_output=True, text=True, cwd=ROOT, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    return json.loads(out.stdout.splitlines()[-1])


@pytest.mark.parametrize("tokens,requests,heads,kv_heads,D,max_q,max_kv", [
    (1, 1, 32, 32, 128, 512, 64), (4, 4, 160, 160, 128, 512, 4096), (2, 1, 8, 1, 64, 4096, 1), (3, 2, 64, 8, 128, 64, 4096),
    (1, 1, 1, 1, 128, 1 << 20, 1 << 18), (600, 2, 32, 32, 128, 512, 600), (7, 1100, 8, 2, 64, 4096, 4096),
])
def test_every_launch_has_workgroups(fake, tokens, requests, heads, kv_heads, D, max_q, max_kv):
    """max_q bounds a request's new tokens and may be far more than there are."""
    (ls,) = launches(fake, [[tokens, requests, heads, kv_heads, D, max_q, max_kv, True]])
    assert ls and all(x["grid"] > 0 for x in ls), ls


@pytest.mark.parametrize("D,g", [(128, -1), (128, 32), (64, -1)])
@pytest.mark.parametrize("heads,kv_heads", [(32, 32), (64, 8), (64, 64), (16, 4), (24, 2), (160, 160), (128, 1)])
def test_plan_names_what_runs(fake, D, g, heads, kv_heads):
    """The plan query against the launches: kernel, workgroups and whether scratch is asked for;
    with a shorter request among them scratch is asked for only where the plan says so."""
    shapes = [(r, n, kv) for r in (1, 2, 17, 64, 1030) for n in (1, 2, 5, 9, 40, 81, 200, 600) for kv in (60, 65, 257, 5000)]
    calls = [[r * n, r, heads, kv_heads, D, n, kv, n > 1, g] for r, n, kv in shapes]
    shorter = [[r * n - n + 1, r, heads, kv_heads, D, n, kv, True, g] for r, n, kv in shapes]
    out = (ctypes.c_int * 3)()
    for (r, n, kv), full, mixed in zip(shapes, launches(fake, calls), launches(fake, shorter)):
        assert _lib.load().marlin_hip_kv4_plan(r, heads, kv_heads, D, g, n, kv, 256, out) == 0
        kernel, workgroups, split = out
        assert full[0]["kernel"] == ("kv4_split_kernel", "kv4_prompt_kernel")[kernel], (r, n, kv)
        assert full[0]["grid"] == workgroups, (r, n, kv, full, list(out))
        assert len(full) == -(-r // 1024)
        asked = any(x["scratch"] for x in full)
        assert asked == bool(split) if kernel == 0 else asked <= split, (r, n, kv, full, list(out))
        assert any(x["scratch"] for x in mixed) <= split, (r, n, kv, mixed, list(out))


def _main(req):
    fake = ctypes.CDLL(req["fake"], mode=ctypes.RTLD_GLOBAL)
    fake.fake_hip_launch.restype = ctypes.c_char_p
    lib = _lib.load()
    if "tables" in req:
        p, (width, page) = ctypes.c_void_p(4096), req["tables"]
        print(lib.marlin_hip_kv4_tables(p, p, p, p, p, p, p, p, 1, 1, width, page, 1, 0, ctypes.c_void_p(64)))
        return
    u, out, seen = [ctypes.c_uint(), ctypes.c_uint(), ctypes.c_int(), ctypes.c_int()], [], 0
    at = ctypes.c_void_p()

    def allocated():  # (the stand-in's allocator only counts up)
        fake.hipMalloc(ctypes.byref(at), ctypes.c_size_t(4096))
        return at.value

    for n, call in enumerate(req["calls"]):
        before = allocated()
        err = attention(lib, 4096, *call, *[-1] * (len(call) == 8), 64 * (n + 1))
        assert err == 0, (call, err, _lib.last_error())
        scratch, mine = allocated() - before > 4096, []
        for i in range(seen, fake.fake_hip_launches()):
            name = fake.fake_hip_launch(i, *map(ctypes.byref, u)).decode()
            mine.append({"kernel": _base(name), "grid": u[0].value, "scratch": scratch})
        seen += len(mine)
        out.append(mine)
    print(json.dumps(out))


if __name__ == "__main__":
    _main(json.loads(sys.argv[1]))
