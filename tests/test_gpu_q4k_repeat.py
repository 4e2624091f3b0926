"""The shared-memory form of the packed Q4_K projection over many launches: the
producers hand a packed slot back while the epilogue of the tile before keeps
the memory pipe busy, so a slot refilled too early shows in some launches only
(before its mend 9 of 65 products of this shape held wrong rows).

TVARA_Q4K_A is read once per process, so the launches run in a child."""

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

CHILD = """
import ctypes as C, sys
import numpy as np, torch
from tvara_b200 import gguf, load_library
lib = load_library()
rows, cols, tokens, launches = map(int, sys.argv[1:])
raw = np.frombuffer(gguf.random_blocks(gguf.Q4_K, rows, cols, np.random.default_rng(7)), np.uint8).copy()
raw = torch.from_numpy(raw).cuda()
at = lambda t: C.c_void_p(t.data_ptr())
buf = torch.empty(lib.tvara_packed_bytes(gguf.Q4_K, rows, cols), dtype=torch.uint8, device="cuda")
assert lib.tvara_pack(gguf.Q4_K, at(raw), rows, cols, at(buf), None) == 0
w = torch.empty(rows, cols, device="cuda")
assert lib.tvara_dequantize(gguf.Q4_K, at(raw), rows * cols // 256, at(w), None) == 0
x = torch.randn(tokens, cols, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
want = x.double() @ w.double().T
bound = 2e-5 * (x.double().abs() @ w.double().abs().T) + 1e-6
size = lib.tvara_quant_matmul_workspace(cols, tokens)
work = torch.empty(size, dtype=torch.uint8, device="cuda")
for i in range(launches):
    y = torch.full((tokens, rows), float("nan"), device="cuda")
    assert lib.tvara_quant_matmul(gguf.Q4_K, at(buf), rows, cols, at(x), tokens, at(y), at(work), size, None) == 0
    assert ((y.double() - want).abs() <= bound).all(), i
"""


@pytest.mark.parametrize("rows,cols,tokens", [(11008, 4096, 512), (4096, 4096, 512)])
def test_shared_memory_form_many_launches(rows, cols, tokens):
    env = dict(os.environ, TVARA_Q4K_A="smem", PYTHONPATH=str(ROOT))
    res = subprocess.run([sys.executable, "-c", CHILD, str(rows), str(cols), str(tokens), "400"], cwd=ROOT, env=env,
                         capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout[-1000:] + res.stderr[-2000:]
