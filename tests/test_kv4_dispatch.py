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


def attention(lib, at, tokens, requests, q_heads, kv_heads, head_dim, max_q, max_kv, cu_q, groupsize=-1):
    """One call with operands at address ``at``, which is never read on the host."""
    p = ctypes.c_void_p(at)
    return lib.marlin_hip_kv4_attention(p, p, p, p, p if cu_q else NULL, p, NULL, tokens, requests, q_heads, kv_heads,
                                        head_dim, q_heads * head_dim, head_dim, 16, 1 << 16, 1 << 14, groupsize, max_q,
                                        max_kv, 1.0, 0, 0, ctypes.c_void_p(64))


def test_one_token_a_request_needs_as_many_tokens(built_lib):
    """Without cu_q request i is token i: fewer tokens than requests would be read past q."""
    assert attention(built_lib, 0, 3, 4, 8, 2, 128, 1, 64, False) == _lib.ERR_PROB_SHAPE
    assert "cu_q" in _lib.last_error()


@pytest.fixture(scope="module")
def fake(built_lib, tmp_path_factory):
    return build_fake(tmp_path_factory.mktemp("fake_hip"))


def launches(fake, calls):
    """Per call (the arguments of ``attention`` after ``at``) its launches, kernel and grid, seen
    in a process of its own."""
    out = subprocess.run([sys.executable, str(pathlib.Path(__file__)), json.dumps({"fake": str(fake), "calls": calls})],
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


def _main(req):
    fake = ctypes.CDLL(req["fake"], mode=ctypes.RTLD_GLOBAL)
    fake.fake_hip_launch.restype = ctypes.c_char_p
    lib = _lib.load()
    u, out, seen = [ctypes.c_uint(), ctypes.c_uint(), ctypes.c_int(), ctypes.c_int()], [], 0
    for call in req["calls"]:
        err = attention(lib, 4096, *call)
        assert err == 0, (call, err, _lib.last_error())
        mine = []
        for i in range(seen, fake.fake_hip_launches()):
            name = fake.fake_hip_launch(i, *map(ctypes.byref, u)).decode()
            mine.append({"kernel": _base(name), "grid": u[0].value})
        seen += len(mine)
        out.append(mine)
    print(json.dumps(out))


if __name__ == "__main__":
    _main(json.loads(sys.argv[1]))
