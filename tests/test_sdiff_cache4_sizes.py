"""Size functions of the C interface over any arguments, on the CPU."""
import subprocess
import sys

from tda_b200 import _lib

GOOD = dict(map=0, batch=2, heads=8, kv_heads=2, head_dim=128, page=64, width=256)
TOP = 2 ** 62
BAD = [
    dict(heads=0), dict(heads=-8), dict(heads=7), dict(heads=1), dict(heads=TOP), dict(kv_heads=0), dict(kv_heads=-2), dict(batch=0),
    dict(batch=-1), dict(batch=TOP), dict(head_dim=0), dict(head_dim=96), dict(page=0), dict(page=-16), dict(page=48),
    dict(width=0), dict(width=-1), dict(width=TOP), dict(heads=0, kv_heads=1, batch=TOP),
]


def test_cache_workspace_of_refused_sizes():
    """0 for each, in a process of its own: a division by zero would end it."""
    code = "from tda_b200 import _lib\nsize = _lib.load().tda_cache4_workspace_size\n"
    code += f"for a in {[tuple({**GOOD, **b}.values()) for b in BAD]}: print(size(*a), flush=True)"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.stdout.split() == ["0"] * len(BAD), (len(r.stdout.split()), r.returncode, r.stderr)
    assert r.returncode == 0


def test_cache_workspace_of_good_sizes():
    size = _lib.load().tda_cache4_workspace_size
    at = lambda **kw: size(*{**GOOD, **kw}.values())
    assert at() > 0 and at() % (2 * 8 * (8 + 2 * 128) * 4) == 0
    assert at(map=1) * (8 + 2 * 128) == at() * 128
    assert at(width=1) == 0  # one chunk: nothing to join
    assert at(batch=65535, heads=64, kv_heads=8, width=1 << 14) > 2 ** 32
