"""The compiled binding of the paged operators: loaded by them alone, one for each Python and torch."""
from __future__ import annotations

import importlib.metadata
import subprocess
import sys
from pathlib import Path

from sparseattentioninfer_b200 import _build

ROOT = Path(__file__).resolve().parents[1]


def test_the_package_works_without_the_binding():
    """The dense operators and the backend import; a paged call says what is missing."""
    code = """
import importlib.util as u
real = u.spec_from_file_location
def absent(name, *a, **k):
    if name == "_sa_paged":
        raise ImportError("no binding")
    return real(name, *a, **k)
u.spec_from_file_location = absent
import torch
import sparseattentioninfer_b200 as sa
sa.get_backend("cuda_sm100")
q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
try:
    sa.ops.paged_attention(q, q, q, q, q, q)
except ImportError as e:
    print(e)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.strip() == "no binding", r.stderr[-2000:]


def test_another_torch_asks_for_another_binding(monkeypatch):
    here = _build.binding_path()
    assert here.exists()
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1")
    assert _build.binding_path() != here and not _build.binding_path().exists() and _build.needs_build()
