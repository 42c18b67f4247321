"""The package without the serving operators' module: everything else imports, and their calls say what is missing."""
import os
import shutil
import subprocess
import sys

import pytest

pytest.importorskip("torch")

import saccade_core as sc

CODE = """
import torch, saccade_core as sc
from saccade_core import qwen2
assert sc.SaccadeLinearOp and qwen2.GreedyDecoder and sc.LIB_PATH
c = sc.PagedKVCache(1, 4, 16, 1, 64, max_seqs=1, max_positions=32, device="cpu")
x = torch.zeros(1, 1, 64)
i = torch.zeros(1, 1, dtype=torch.int32)
for call in (lambda: sc.process_logits(torch.zeros(1, 4)),
             lambda: sc.paged_append(x, x, x, x[0], x[0], c.k[0], c.v[0], i, i[0], i[0]),
             lambda: sc.paged_attention(x, c.k[0], c.v[0], i, i[0], i[0], 1, 1)):
    try:
        call()
    except ImportError as e:
        assert "make -C csrc" in str(e) and e.__cause__ is not None, e
    else:
        raise AssertionError("no module, but an answer")
print("ok")
"""


@pytest.mark.parametrize("how", ["absent", "broken"])
def test_the_package_without_the_module(tmp_path, how):
    src = os.path.dirname(sc.__file__)
    dst = tmp_path / "saccade_core"
    shutil.copytree(src, dst, ignore=shutil.ignore_patterns("_serve*", "__pycache__"))
    if how == "broken":
        (dst / "_serve.so").write_bytes(b"no shared object")
    env = dict(os.environ, PYTHONPATH=str(tmp_path), SACCADE_CTARQ_LIB=sc.LIB_PATH)
    r = subprocess.run([sys.executable, "-c", CODE], env=env, cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr


def test_here_the_module_is_there():
    from saccade_core import _serve, paged
    assert paged._serve is _serve
