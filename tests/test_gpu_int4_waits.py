"""Waits of ``int4_mma_kernel`` that run out: the kernel sets the status word, writes nothing more, waits for what it has
started, and leaves the GPU as usable as before.  Here its copies of x stop after some steps (``c_abi/int4_waits.cu``)."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def waits(tmp_path_factory):
    from flashsampling_b200 import build

    build.build_library()
    out = tmp_path_factory.mktemp("waits") / "libint4_waits.so"
    cmd = [build._nvcc(), *build.NVCC_FLAGS, "-I", str(build.CSRC), "-o", str(out), str(ROOT / "tests" / "c_abi" / "int4_waits.cu")]
    done = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]
    fn = ctypes.CDLL(str(out)).int4_with_x_limit
    p, i, u = ctypes.c_void_p, ctypes.c_int, ctypes.c_ulonglong
    fn.argtypes = [p, p, p, i, i, i, p, p, u, p, u, i, p]
    return fn


# columns in steps of 256; 2048 rows: one tile per CTA, 21400 rows: up to ten, in two blocks of eight
@pytest.mark.parametrize("rows,cols,limit", [(2048, 4096, 0), (2048, 4096, 1), (2048, 4096, 2), (2048, 4096, 3), (2048, 4096, 9), (2048, 4096, 15),
                                             (21400, 1024, 3), (21400, 1024, 4), (21400, 1024, 6), (21400, 1024, 8)])
def test_a_wait_that_runs_out(waits, rows, cols, limit):
    import flashsampling_b200 as fs
    from flashsampling_b200 import _lib

    dev, batch = torch.device("cuda", 0), 12
    g = torch.Generator().manual_seed(rows)
    w = fs.Int4Weight.from_rows(torch.randint(0, 16, (rows, cols), generator=g, dtype=torch.uint8).to(dev),
                                (torch.rand(rows, cols // 128, generator=g) * 0.01).bfloat16().to(dev))
    x = torch.randn(batch, cols, generator=g).bfloat16().to(dev)
    want = fs.int4_linear(x, w, out_dtype=torch.float32)
    ws = torch.empty(_lib.query_int4_workspace(rows, cols, 128, batch), dtype=torch.uint8, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)

    def call(limit):
        out = torch.full((batch, rows), 7.0, device=dev)
        rc = waits(x.data_ptr(), w.qweight.data_ptr(), w.scales.data_ptr(), rows, cols, batch, out.data_ptr(), ws.data_ptr(), ws.numel(),
                   status.data_ptr(), 50_000_000, limit, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        return out

    steps = cols // 256
    tiles = -(-rows // 16)
    per_cta = -(-tiles // torch.cuda.get_device_properties(dev).multi_processor_count)
    out = call(limit)
    written = out != 7
    if limit >= steps * -(-per_cta // 8):
        assert int(status.item()) == 0 and torch.equal(out, want)
    else:
        assert int(status.item()) == _lib.ERR_TIMEOUT
        assert torch.equal(out[written], want[written])  # what is there is right, the rest as it was
        assert bool(written.any()) == (limit >= steps)
    status.zero_()
    assert torch.equal(call(1 << 30), want) and int(status.item()) == 0
    assert torch.equal(fs.int4_linear(x, w, out_dtype=torch.float32), want)
    fs.check_status()
