"""The generator with its backbone cache in 8 bits reports what goes wrong on the device (needs a B200): prompts and steps
whose attention gives up raise, the session of a failed prompt is gone, and the generator stays usable. In a
process of its own, as the cache's type is read from the environment."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_SCRIPT = r"""
import sys
import numpy as np
sys.path.insert(0, sys.argv[1])
import __graft_entry__ as g
pkg = g.load_package()
rng = np.random.default_rng(11)
text = lambda n: pkg.ids_to_text(rng.integers(300, 20000, n).tolist())

def fails(f):
    try:
        f()
    except RuntimeError as e:
        assert "8-bit cache" in str(e) and "timed out" in str(e), str(e)
        return
    raise SystemExit("no error was raised")

words = [text(n) for n in (40, 150, 33)]
gen = pkg.GeneratorHandle(sys.argv[2], 0)
specs = [dict(session_id=50 + i, text=words[i], seed=i, max_new_tokens=9) for i in range(2)]
pkg.set_debug_kv8_polls(0)
fails(lambda: gen.sessions_create_batch(specs))
fails(lambda: gen.session_create_ext(80, words[2], seed=7, max_new_tokens=9))
pkg.set_debug_kv8_polls(-1)
assert gen.active_session_count() == 0
# the words were cleared, and the same prompts succeed
gen.sessions_create_batch(specs)
gen.session_create_ext(80, words[2], seed=7, max_new_tokens=9)
assert gen.active_session_count() == 3
# a step's graph keeps the limit that it was captured with
pkg.set_debug_kv8_polls(0)
fails(lambda: gen.step_frames([50, 80], 1, [1, 2]))
gen.close()
pkg.set_debug_kv8_polls(-1)
gen = pkg.GeneratorHandle(sys.argv[2], 0)
gen.session_create_ext(80, words[2], seed=7, max_new_tokens=9)
n, frames, _ = gen.step_frames([80], 2, [1])
assert n == 2 and (frames[:, 0, 0] >= 0).all()
gen.close()
print("reported")
"""


def test_attention_that_gives_up_is_an_error_of_the_call(tiny_model):
    r = subprocess.run([sys.executable, "-c", _SCRIPT, ROOT, tiny_model],
                       env=dict(os.environ, BZB_KV_CACHE="e4m3", BZB_KV8_ATTENTION="many"), capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "reported" in r.stdout, r.stdout[-1000:] + r.stderr[-2000:]
