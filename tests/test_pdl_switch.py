"""Programmatic dependent launch inside a call (layer norm, gated feed-forward): what switches it, and that results do not depend on it."""
import hashlib
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code, **env):
    e = {k: v for k, v in os.environ.items() if k not in ("CHOCO_PDL", "CHOCO_PDL_CALLS")}
    r = subprocess.run([sys.executable, "-c", code], env=dict(e, **env), cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr
    return r.stdout.strip()


_ASK = """
import os, torch
from chocosgd_b200 import build_ext
from chocosgd_b200.ops import _lib
build_ext.build()
for env, mode, bf16 in CASES:
    r, w = os.pipe()
    if os.fork() == 0:                    # the switches are read once per process
        os.environ.update(env)
        if mode:
            _lib.configure_pdl(mode, bf16=bf16)
        os.write(w, str(_lib.load().choco_pdl_in_call()).encode())
        os._exit(0)
    print(os.read(r, 1).decode(), end="")
"""


def test_switches():
    cases = [({}, "", False, "1"), ({"CHOCO_PDL": "0"}, "", False, "0"), ({"CHOCO_PDL": "1"}, "", False, "1"),
             ({"CHOCO_PDL_CALLS": "0"}, "", False, "0"), ({"CHOCO_PDL": "0", "CHOCO_PDL_CALLS": "1"}, "", False, "1"),
             ({"CHOCO_PDL": "1", "CHOCO_PDL_CALLS": "0"}, "", False, "1"),
             ({}, "auto", False, "1"), ({}, "auto", True, "1"), ({}, "on", False, "1"), ({}, "off", False, "0"), ({}, "off", True, "0"),
             ({"CHOCO_PDL": "0"}, "auto", False, "0"),            # an explicit environment setting wins
             ({"CHOCO_PDL_CALLS": "1"}, "off", False, "1")]
    got = _run(_ASK.replace("CASES", repr([c[:3] for c in cases])))
    assert got == "".join(c[3] for c in cases)


_BLOCK = """
import hashlib, torch
from chocosgd_b200.ops.ffn import gated_ffn
from chocosgd_b200.ops.norm import layer_norm
h = hashlib.sha256()
for dtype in (torch.float32, torch.bfloat16):
    for m in (1, 12, 300):
        g = torch.Generator(device="cuda").manual_seed(m)
        leaves = [torch.randn(*s, device="cuda", generator=g).mul_(0.2).to(dtype).requires_grad_() for s in ((m, 70), (70,), (272, 70), (70, 136))]
        dy = torch.randn(m, 70, device="cuda", generator=g).to(dtype)
        for _ in range(3):
            y = gated_ffn(layer_norm(*leaves[:2]), *leaves[2:])
            outs = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
            with torch.no_grad():
                outs.append(gated_ffn(layer_norm(*leaves[:2]), *leaves[2:]))
        for t in outs:
            h.update(t.float().cpu().numpy().tobytes())
print(h.hexdigest())
"""


@pytest.mark.gpu
def test_the_same_bits_with_and_without():
    want = _run(_BLOCK)
    assert len(want) == len(hashlib.sha256().hexdigest())
    for env in ({"CHOCO_PDL": "0"}, {"CHOCO_PDL": "1"}):
        assert _run(_BLOCK, **env) == want
