"""How attention behind shared prefixes is launched, on the CPU: the plan query against the launches of the call
(tests/fake_hip.cpp stands in for the HIP runtime), and the rules for two passes and for parts left to the second."""
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

# requests, new tokens of each, groups, query heads, kv heads, head dim, max_kv
SHAPES = [(r, n, g, *h, kv) for r in (2, 64, 1100) for n in (1, 4, 100) for g in (1, 4, 2000)
          for h in ((32, 32, 128), (64, 8, 128), (16, 4, 64), (300, 300, 128)) for kv in (60, 16384)]


def plan(lib, r, n, g, hq, h, d, kv, always, group=-1, most=None):
    out = (ctypes.c_longlong * 3)()
    assert lib.marlin_hip_kv4_shared_plan(r * n, r, g, hq, h, d, group, n if most is None else most, kv, n > 1, always, -1, out) == 0
    return list(out)


@pytest.fixture(scope="module")
def ran(built_lib, tmp_path_factory):
    """Per shape, without and with ``always``: the launches of the call with the workspace that the plan names, the
    code with four bytes less than two passes need, and that with just those."""
    fake = build_fake(tmp_path_factory.mktemp("fake_hip"))
    out = subprocess.run([sys.executable, str(pathlib.Path(__file__)), str(fake)], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    return json.loads(out.stdout.splitlines()[-1])


def test_plan_is_what_runs(built_lib, ran):
    kinds = set()
    for (shape, always), (code, launches, short, least) in zip(((s, a) for s in SHAPES for a in (0, 1)), ran):
        size, prompts, parts = plan(built_lib, *shape, always)
        r, n, g, hq, h, d, kv = shape
        assert code == _lib.OK and launches and size % 4 == 0
        if size == 0:  # plain attention, no workspace
            assert not always and all(form == 0 for _, form in launches) and short == least == _lib.OK
            continue
        assert all(form == 1 for _, form in launches)
        assert launches[0][0] == ("kv4_split_kernel", "kv4_prompt_kernel")[prompts], (shape, always)
        assert all(k == launches[0][0] for k, _ in launches[:-(-g // 1024)])
        need = 4 * r * n * hq * (d + 2)
        assert size >= need and (size == need) == (not parts)
        if parts:  # the rows, where their parts lie, and 256 rows a compute unit
            places = 256 // h * h * 256
            assert prompts and g <= 1024 and 0 <= size - 4 * (r * n * hq * (d + 4) + places * (d + 2)) < 16
        assert short == _lib.ERR_PROB_SHAPE and least == _lib.OK
        kinds.add((always, prompts, parts))
    assert kinds == {(a, *k) for a in (0, 1) for k in ((0, 0), (1, 0), (1, 1))}


def test_two_passes_where_more_reads_fall_away(built_lib):
    """Monotonous in the prefix and in the requests of a group; none where nothing is shared; ``always`` whatever the sizes."""
    for n, hq, h, d in ((1, 32, 32, 128), (1, 64, 8, 128), (4, 32, 32, 128), (300, 64, 8, 128)):
        by_len = [plan(built_lib, 16, n, 1, hq, h, d, kv, 0)[0] > 0 for kv in (0, 64, 500, 4000, 30000, 1 << 20)]
        by_requests = [plan(built_lib, r, n, 1, hq, h, d, 4096, 0)[0] > 0 for r in (1, 2, 8, 64, 512)]
        assert by_len == sorted(by_len) and by_requests == sorted(by_requests) and by_len[-1] and not by_len[0] and not by_requests[0]
        assert plan(built_lib, 16, n, 16, hq, h, d, 1 << 20, 0)[0] == 0
        assert plan(built_lib, 1, n, 1, hq, h, d, 64, 1)[0] > 0
    # the sides that were measured
    for r, n, g, hq, h, kv, two in ((16, 1, 1, 64, 8, 8192, False), (32, 1, 4, 32, 32, 1600, True), (32, 1, 1, 32, 32, 4200, True),
                                    (8, 1, 1, 64, 8, 8200, False), (64, 1, 1, 64, 8, 8400, True), (4, 200, 1, 32, 32, 400, False)):
        assert (plan(built_lib, r, n, g, hq, h, 128, kv, 0)[0] > 0) == two, (r, n, g, hq, h, kv)


def test_refusals_and_nothing_to_do(built_lib):
    out = (ctypes.c_longlong * 3)(7, 7, 7)
    ask = lambda tokens=4, requests=4, groups=1, hq=8, h=2, d=128, g=-1, q=1, kv=64: built_lib.marlin_hip_kv4_shared_plan(  # noqa: E731
        tokens, requests, groups, hq, h, d, g, q, kv, 0, 1, -1, out)
    for change in ({"tokens": 0}, {"requests": 0}, {"groups": 0}, {"q": 0}):
        out[0] = 7
        assert ask(**change) == _lib.OK and list(out) == [0, 0, 0]
    for change in ({"tokens": -1}, {"requests": -1}, {"groups": -1}, {"groups": 2 ** 20 + 1}, {"hq": 9}, {"h": 0}, {"q": -1}, {"kv": -1}):
        assert ask(**change) == _lib.ERR_PROB_SHAPE, change
    for change in ({"d": 96}, {"g": 16}):
        assert ask(**change) == _lib.ERR_KERN_SHAPE


def _main(fake_lib):
    fake = ctypes.CDLL(fake_lib, mode=ctypes.RTLD_GLOBAL)
    fake.fake_hip_launch.restype = ctypes.c_char_p
    lib = _lib.load()
    p, null, u = ctypes.c_void_p(4096), ctypes.c_void_p(0), [ctypes.c_uint(), ctypes.c_uint(), ctypes.c_int(), ctypes.c_int()]

    def call(r, n, g, hq, h, d, kv, always, size):
        return lib.marlin_hip_kv4_attention_shared(p, p, p, p, p if n > 1 else null, p, p, p, null, p if size else null, r * n, r, g, hq, h,
                                                   d, hq * d, d, 16, 1 << 16, 1 << 14, -1, n, kv, 1.0, 0, size, always, 0, ctypes.c_void_p(64))

    out, seen = [], 0
    for shape in SHAPES:
        for always in (0, 1):
            size = plan(lib, *shape, always)[0]
            code, mine = call(*shape, always, size), []
            for i in range(seen, fake.fake_hip_launches()):
                name = fake.fake_hip_launch(i, *map(ctypes.byref, u)).decode()
                mine.append((_base(name), int(name.split("EEE")[0][-1])))  # (the last template argument)
            need = 4 * shape[0] * shape[1] * shape[3] * (shape[5] + 2) if size else 0
            out.append((code, mine, call(*shape, always, max(need - 4, 0)), call(*shape, always, need)))
            seen = fake.fake_hip_launches()
    print(json.dumps(out))


if __name__ == "__main__":
    _main(sys.argv[1])
