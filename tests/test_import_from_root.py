"""A program started in the repository's root, with nothing set, imports the
package (it lies in vosk-api_amd/); one that has put vosk-api_amd/ on its path
gets the same files.  CPU-only: importing loads libvosk.so and touches no
device."""
import os
import subprocess
import sys

import pytest

from conftest import PKG, REPO

ORDERS = {"the root alone": [], "the package's folder behind the root": [None, PKG], "ahead of it": [PKG, None]}


def _run(code, tmp_path, path=()):
    env = {k: v for k, v in os.environ.items() if k not in ("PYTHONPATH", "PYTHONSAFEPATH")}
    env["PYTHONDONTWRITEBYTECODE"] = "1"
    if path:
        env["PYTHONPATH"] = os.pathsep.join(p or REPO for p in path)
    out = subprocess.run([sys.executable, "-c", code], cwd=REPO if not path else tmp_path, env=env, capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    return out.stdout.split("\n")[:-1]


@pytest.mark.parametrize("path", ORDERS.values(), ids=ORDERS.keys())
def test_package_and_its_modules(path, tmp_path):
    got = _run("import torch\nfrom vosk import ops\nimport vosk, vosk.engine, sys\n"
               "print(vosk.__file__, ops.__file__, vosk.engine.__file__, sep='\\n')\n"
               "print(sys.modules['vosk'] is vosk and vosk.ops is ops and vosk.ops._c is vosk._c is vosk.engine._c)\n"
               "print(vosk.__name__, vosk.KaldiRecognizer.__module__)", tmp_path, path)
    want = [os.path.join(PKG, "vosk", f) for f in ("__init__.py", "ops.py", "engine.py")]
    assert [os.path.realpath(f) for f in got[:3]] == [os.path.realpath(f) for f in want]
    assert got[3:] == ["True", "vosk vosk"]


def test_a_failing_import_can_be_tried_again(tmp_path):
    """A library that is not there: OSError as from the package's own folder, and nothing half-imported stays."""
    got = _run("import os, sys\nos.environ['VOSK_AMD_LIB'] = '/nowhere/libvosk.so'\n"
               "try:\n    import vosk\nexcept OSError as e:\n    print('/nowhere' in str(e), 'vosk' in sys.modules)\n"
               "del os.environ['VOSK_AMD_LIB']\nimport vosk\nprint(hasattr(vosk, 'Model'))", tmp_path)
    assert got == ["True False", "True"]


def test_two_threads_import_it(tmp_path):
    """The second waits until the package is whole."""
    got = _run("import sys, threading\nseen = []\n"
               "def go():\n    import vosk\n    seen.append(hasattr(vosk, 'BatchRecognizer'))\n"
               "sys.setswitchinterval(1e-5)\nts = [threading.Thread(target=go) for _ in range(8)]\n"
               "[t.start() for t in ts]\n[t.join() for t in ts]\nprint(seen.count(True), len(seen))", tmp_path)
    assert got == ["8 8"]
