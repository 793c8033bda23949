"""The shared pool of cached keys and values on the device, at the ends of what its calls allow."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

# ------------------------------------------------------------------------------------------------ wide tables
WIDE_TABLES = """
import sys
import numpy as np, torch
import kronos_2t_b200 as k2
d = int(sys.argv[1])
ctx = k2.Context(0)
ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
pool = k2.KvPool(ctx, 1, d, 8, 16, 64, block_keys=True)
rng = np.random.default_rng(0)
k = torch.from_numpy(rng.standard_normal((640, 1, d)).astype(np.float32)).cuda()
pool.store_dev("f32", k.data_ptr(), k.data_ptr(), torch.arange(640, device="cuda").data_ptr(), 640)
q = torch.from_numpy(rng.standard_normal((1, 1, d)).astype(np.float32)).cuda()
lens = torch.tensor([640], dtype=torch.int32, device="cuda")
want = None
for width in (40, 4096, 4097, 9788, 9789, 10240, 10892, 10893, 12287, 12288, 12289, 20000, 32768):
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, :40] = torch.arange(40)
    out = torch.full((1, 1, 9), 77, dtype=torch.int32, device="cuda")
    pool.select_dev("f32", 1, 1, q.data_ptr(), lens.data_ptr(), table.data_ptr(), width, 9, out.data_ptr(), sinks=1, local=1)
    ctx.synchronize()
    got = out.cpu().tolist()
    want = want or got
    assert got == want and got[0][0][0] == 0 and got[0][0][-1] == 39, (width, got, want)
print("widths agree")
"""

@pytest.mark.parametrize("d", [64, 128])
def test_choice_in_tables_of_every_width(d):
    """The table's width alone sizes the kernel's shared memory; in a process of its own, widths ascending, so that no wider call has gone before."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, "-c", WIDE_TABLES, str(d)], cwd=root, capture_output=True, text=True, timeout=600)
    assert got.returncode == 0 and "widths agree" in got.stdout, got.stderr[-2000:]
