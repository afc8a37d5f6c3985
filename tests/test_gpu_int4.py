"""4-bit products against the dequantised weight in 64 bits.

Tolerance.  Every product of a code (4 bits) with an x in fp16 is exact.  x reaches fp16 after a power of two that puts
its row's maximum at 2^14 or above, from nine rows on at 2^7 or above: where bits are lost, half a step of the smallest
fp16 numbers is 2^-25, or 2^-39 and 2^-32 of that maximum.  What rounds are fp32 additions.  Tensor cores may
truncate (2^-23 relative to the largest partial sum) and every partial sum is at most A = sum_k scale (q + zero) |x|.  An
output passes through at most 16 additions inside a product, group / 16 products, cols / group group sums, 16 warps, 8
CTAs, and 8 further roundings (sums of x, zero point, scales, powers of two): error <= n 2^-23 A with that n.  The
output type adds half a step: eps / 2 relative.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fs():
    import flashsampling_b200 as fs
    from flashsampling_b200 import build

    build.build_library()
    return fs


def _dev():
    return torch.device("cuda", 0)


def _weight(fs, rows, cols, group, zeros, seed=0, scale_dtype=torch.bfloat16):
    g = torch.Generator(device=_dev()).manual_seed(seed)
    q = torch.randint(0, 16, (rows, cols), generator=g, device=_dev(), dtype=torch.uint8)
    s = ((torch.rand(rows, cols // group, generator=g, device=_dev()) + 0.5) * 0.01).to(scale_dtype)
    z = torch.randint(0, 16, (rows, cols // group), generator=g, device=_dev(), dtype=torch.uint8) if zeros else None
    return fs.Int4Weight.from_rows(q, s, z)


def _x(batch, cols, dtype, seed=1):
    g = torch.Generator(device=_dev()).manual_seed(seed)
    x = torch.randn(batch, cols, generator=g, device=_dev())
    x[:, ::97] *= 30
    return x.to(dtype)


def _reference(w, x):
    """The result in 64 bits and the bound of its computation in 32."""
    wd = w.dequantize(torch.float64)
    scale = w.scales.permute(0, 3, 2, 1).reshape(-1, w.scales.shape[1])[:w.rows].double().repeat_interleave(w.group_size, 1)
    zero = 8.0 if w.zeros is None else w.zeros.permute(0, 3, 2, 1).reshape(-1, w.scales.shape[1])[:w.rows].double().repeat_interleave(w.group_size, 1)
    xd = x.double().reshape(-1, w.cols)
    amount = xd.abs() @ (scale.abs() * (w.codes().double() + zero)).T
    n = 16 + w.group_size // 16 + w.cols // w.group_size + 16 + 8 + 8
    tiny = xd.abs().amax(1, keepdim=True) * (2.0**-39 if xd.shape[0] <= 8 else 2.0**-32) * (scale.abs() * 16).sum(1)
    shape = x.shape[:-1] + (w.rows,)
    return (xd @ wd.T).view(shape), (n * 2.0**-23 * amount + tiny).view(shape)


def _check(y, want, bound):
    tol = bound + want.abs() * torch.finfo(y.dtype).eps / 2 + torch.finfo(y.dtype).tiny
    over = (y.double() - want).abs() > tol
    assert not bool(over.any()), f"{int(over.sum())} of {over.numel()} outputs off, worst {float(((y.double() - want).abs() / tol).max()):.2f} of the bound"


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("rows,cols,batch", [(1, 256, 1), (16, 256, 1), (17, 512, 3), (100, 1024, 8), (250, 768, 9),
                                              (333, 2048, 16), (64, 4352, 17), (2500, 1280, 32), (75, 512, 70)])
def test_against_the_dequantised_weight(fs, rows, cols, batch, group, zeros):
    w = _weight(fs, rows, cols, group, zeros, seed=rows + group)
    x = _x(batch, cols, torch.bfloat16, seed=cols)
    want, bound = _reference(w, x)
    _check(fs.int4_linear(x, w, out_dtype=torch.float32), want, bound)
    fs.check_status()


@pytest.mark.parametrize("cols,group", [(640, 640), (2688, 384), (5376, 2688), (9216, 512)])
def test_groups_of_many_columns(fs, cols, group):
    w = _weight(fs, 170, cols, group, True, seed=cols)
    x = _x(9, cols, torch.bfloat16)
    want, bound = _reference(w, x)
    _check(fs.int4_linear(x, w, out_dtype=torch.float32), want, bound)


@pytest.mark.parametrize("cols", [64, 192, 320])
def test_half_filled_last_fetch(fs, cols):
    w = _weight(fs, 70, cols, 64, True, seed=cols)
    x = _x(3, cols, torch.bfloat16)
    want, bound = _reference(w, x)
    _check(fs.int4_linear(x, w, out_dtype=torch.float32), want, bound)


@pytest.mark.parametrize("cols", [32, 96, 160, 4128])
def test_half_filled_last_chunk(fs, cols):
    w = _weight(fs, 130, cols, 32, True, seed=cols)
    x = _x(5, cols, torch.float16)
    want, bound = _reference(w, x)
    _check(fs.int4_linear(x, w, out_dtype=torch.float32), want, bound)


@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("st", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ot", [torch.bfloat16, torch.float16, torch.float32, None])
def test_types(fs, xt, st, ot):
    w = _weight(fs, 200, 640, 64, True, scale_dtype=st)
    x = _x(4, 640, xt)
    y = fs.int4_linear(x, w, out_dtype=ot)
    assert y.dtype == (ot or xt)
    _check(y, *_reference(w, x))


@pytest.mark.parametrize("rows,cols,batch,group", [
    (40, 16384, 1, 128),  # few tiles, long rows
    (40, 16384, 16, 128),
    (9000, 8192, 16, 128),  # x of 16 rows does not fit one CTA
    (3000, 16384, 30, 64),
    (500, 28672, 8, 256),
    (48, 65536, 9, 256),
    (16, 256 * 1024, 1, 256),
])
def test_columns_in_phases(fs, rows, cols, batch, group):
    w = _weight(fs, rows, cols, group, True, seed=rows)
    x = _x(batch, cols, torch.bfloat16)
    want, bound = _reference(w, x)
    _check(fs.int4_linear(x, w, out_dtype=torch.float32), want, bound)
    fs.check_status()


@pytest.mark.parametrize("rows,cols,batch", [(151936, 4096, 1), (32776, 5376, 5), (16032, 8192, 12)])
def test_heads(fs, rows, cols, batch):
    w = _weight(fs, rows, cols, 128, True, seed=3)
    x = _x(batch, cols, torch.bfloat16)
    y = fs.int4_linear(x, w, out_dtype=torch.float32)
    at = torch.cat([torch.arange(0, 64), torch.randint(0, rows, (4000,), generator=torch.Generator().manual_seed(0)), torch.arange(rows - 64, rows)])
    q, at = w.codes(), at.to(_dev())
    s = w.scales.permute(0, 3, 2, 1).reshape(-1, w.scales.shape[1])[:rows]
    z = w.zeros.permute(0, 3, 2, 1).reshape(-1, w.scales.shape[1])[:rows]
    part = fs.Int4Weight.from_rows(q[at].contiguous(), s[at].contiguous(), z[at].contiguous())
    want, bound = _reference(part, x)
    _check(y[:, at], want, bound)


def test_magnitudes_of_x(fs):
    """Each row is scaled by itself: rows of 1e-30 and of 1e30 beside each other, and small values beside large ones."""
    w = _weight(fs, 64, 512, 128, True)
    x = _x(8, 512, torch.bfloat16)
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3] = 0
    x[4, 0] = 3e30
    x[5] = torch.finfo(torch.bfloat16).tiny
    x[6] = 0
    x[6, 77] = 1
    want, bound = _reference(w, x)
    y = fs.int4_linear(x, w, out_dtype=torch.float32)
    _check(y, want, bound)
    assert bool((y[3] == 0).all())
    h = _x(3, 512, torch.float16)
    h[0] = torch.finfo(torch.float16).max
    h[1] = 2.0**-24
    _check(fs.int4_linear(h, w, out_dtype=torch.float32), *_reference(w, h))


def test_rows_that_are_not_finite_stay_alone(fs):
    w = _weight(fs, 64, 512, 128, False)
    x = _x(4, 512, torch.bfloat16)
    clean = fs.int4_linear(x, w, out_dtype=torch.float32)
    x[1, 5] = float("nan")
    x[3, 9] = float("inf")
    y = fs.int4_linear(x, w, out_dtype=torch.float32)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[2], clean[2])
    assert not bool(y[1].isfinite().any()) and not bool(y[3].isfinite().any())


def test_strided_and_unaligned_x_and_out(fs):
    w = _weight(fs, 300, 512, 128, True)
    wide = _x(6, 2 * 512 + 3, torch.bfloat16)
    for x in (wide[:, 1:513], wide[:, 8:520], wide[::2, 3:515], wide[:, 0:1024:2], wide[:1, 5:517]):
        _check(fs.int4_linear(x, w, out_dtype=torch.float32), *_reference(w, x))
    x = _x(6, 512, torch.bfloat16)
    want, bound = _reference(w, x)
    buf = torch.full((6, 777), 7.0, device=_dev())
    y = fs.int4_linear(x, w, out=buf[:, 100:400])
    assert y.data_ptr() == buf[:, 100:].data_ptr()
    _check(buf[:, 100:400], want, bound)
    assert bool((buf[:, :100] == 7).all()) and bool((buf[:, 400:] == 7).all())  # nothing else is written


def test_leading_dimensions_and_empty_batch(fs):
    w = _weight(fs, 100, 256, 64, False)
    x = _x(6, 256, torch.float16)
    flat = fs.int4_linear(x, w)
    assert torch.equal(fs.int4_linear(x.view(2, 3, 256), w), flat.view(2, 3, 100))
    assert torch.equal(fs.int4_linear(x[2], w), flat[2])
    assert fs.int4_linear(x[:0], w).shape == (0, 100)
    out = torch.empty(2, 3, 100, dtype=torch.float16, device=_dev())
    assert fs.int4_linear(x.view(2, 3, 256), w, out=out) is out and torch.equal(out.view(6, 100), flat)


def test_same_bits_every_time_and_in_every_batch(fs):
    w = _weight(fs, 3333, 4096, 128, True)
    x = _x(8, 4096, torch.bfloat16)
    first = fs.int4_linear(x, w, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(fs.int4_linear(x, w, out_dtype=torch.float32), first)
    for b in range(8):
        assert torch.equal(fs.int4_linear(x[b:b + 1], w, out_dtype=torch.float32)[0], first[b])


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("batch", [33, 48, 49, 64, 65, 130])
def test_many_rows_of_x(fs, batch, group, zeros):
    """One pass of every width and several, rows that end inside a tile, columns that end inside a step."""
    w = _weight(fs, 150 * 16 + 5, 896, group, zeros, seed=batch)
    x = _x(batch, 896, torch.bfloat16, seed=group)
    want, bound = _reference(w, x)
    _check(fs.int4_linear(x, w, out_dtype=torch.float32), want, bound)
    fs.check_status()


@pytest.mark.parametrize("group", [32, 64, 128, 384])
def test_same_bits_in_every_larger_batch(fs, group):
    w = _weight(fs, 2601, 1152, group, True, seed=group)
    x = _x(130, 1152, torch.bfloat16)
    first = fs.int4_linear(x, w, out_dtype=torch.float32)
    for b in (9, 16, 17, 32, 33, 48, 64, 65, 128):
        assert torch.equal(fs.int4_linear(x[:b], w, out_dtype=torch.float32), first[:b]), b
        assert torch.equal(fs.int4_linear(x[130 - b:], w, out_dtype=torch.float32), first[130 - b:]), b


@pytest.mark.parametrize("cols,group", [(32, 32), (96, 32), (4128, 32), (64, 64), (192, 64), (320, 64), (128, 128), (384, 384)])
@pytest.mark.parametrize("batch", [10, 64])
def test_larger_batches_with_half_filled_steps(fs, batch, cols, group):
    w = _weight(fs, 1200, cols, group, True, seed=cols)
    x = _x(batch, cols, torch.float16)
    want, bound = _reference(w, x)
    _check(fs.int4_linear(x, w, out_dtype=torch.float32), want, bound)


@pytest.mark.parametrize("batch", [4, 12])
def test_scales_far_from_one(fs, batch):
    """Scales at the ends of bf16 with rows of x at the other: the result is in range, and so is every step to it."""
    w = _weight(fs, 48, 256, 64, True)
    x = _x(batch, 256, torch.bfloat16)
    for up in (110, -60):
        scaled = fs.Int4Weight(w.qweight, (w.scales.float() * 2.0**up).bfloat16(), w.zeros, w.rows, w.cols)
        rows = (x.float() * 2.0**-up).bfloat16()
        want, bound = _reference(scaled, rows)
        _check(fs.int4_linear(rows, scaled, out_dtype=torch.float32), want, bound)


@pytest.mark.parametrize("batch", [1, 8, 16, 50])
def test_zero_points_of_all_bytes(fs, batch):
    """A zero point is a byte, not a code: fp16 holds 16 z exactly up to 255."""
    g = torch.Generator(device=_dev()).manual_seed(0)
    q = torch.randint(0, 16, (256, 512), generator=g, device=_dev(), dtype=torch.uint8)
    z = torch.arange(256, device=_dev(), dtype=torch.uint8)[:, None].expand(256, 8).contiguous()
    w = fs.Int4Weight.from_rows(q, torch.full((256, 8), 0.01, device=_dev()).bfloat16(), z)
    x = _x(batch, 512, torch.bfloat16)
    _check(fs.int4_linear(x, w, out_dtype=torch.float32), *_reference(w, x))


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("batch", [2, 24])
def test_a_row_of_the_weight_anywhere(fs, batch, group):
    """The two nibbles of a byte are rows of equal standing, and so are the rows of a tile: what a weight's row gives does
    not depend on where it lies, in a weight so small that its tiles are all split alike.  (Codes in the lowest bits of an fp16 number lost some of their products' bits.)"""
    w = _weight(fs, 160, 512, group, True, seed=9)
    q = w.codes()
    s = w.scales.permute(0, 3, 2, 1).reshape(160, -1)
    z = w.zeros.permute(0, 3, 2, 1).reshape(160, -1)
    x = _x(batch, 512, torch.bfloat16)
    y = fs.int4_linear(x, w, out_dtype=torch.float32)
    for shift in (1, 4, 8, 16, 77):
        at = (torch.arange(160, device=_dev()) + shift) % 160
        moved = fs.Int4Weight.from_rows(q[at].contiguous(), s[at].contiguous(), z[at].contiguous())
        assert torch.equal(fs.int4_linear(x, moved, out_dtype=torch.float32), y[:, at])


@pytest.mark.parametrize("batch", [12, 40])
def test_larger_batches_on_streams_and_in_graphs(fs, batch):
    w = _weight(fs, 3000, 1024, 128, True)
    xs = [_x(batch, 1024, torch.bfloat16, seed=s) for s in range(3)]
    want = [fs.int4_linear(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for s, x in zip(streams, xs):
        with torch.cuda.stream(s):
            got.append([fs.int4_linear(x, w) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(y, e) for ys, e in zip(got, want) for y in ys)
    static = xs[0].clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = fs.int4_linear(static, w)
        graphs.append((g, y))
    for x, e in zip(xs, want):
        static.copy_(x)
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, e) for _, y in graphs)
    fs.check_status()


def test_streams_and_graphs(fs):
    w = _weight(fs, 2000, 2048, 64, True)
    xs = [_x(3, 2048, torch.bfloat16, seed=s) for s in range(4)]
    want = [fs.int4_linear(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for s, x in zip(streams, xs):
        with torch.cuda.stream(s):
            got.append([fs.int4_linear(x, w) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(y, e) for ys, e in zip(got, want) for y in ys)
    static = xs[0].clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = fs.int4_linear(static, w)
        graphs.append((g, y))
    for x, e in zip(xs, want):
        static.copy_(x)
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):  # both at once, on streams of their own
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, e) for _, y in graphs)
    fs.check_status()


def test_refusals(fs):
    w = _weight(fs, 64, 256, 64, False)
    x = _x(2, 256, torch.bfloat16)
    with pytest.raises(TypeError):
        fs.int4_linear(x.float(), w)
    with pytest.raises(ValueError):
        fs.int4_linear(x[:, :128], w)
    with pytest.raises(RuntimeError):
        fs.int4_linear(x.cpu(), w)
    with pytest.raises(RuntimeError):
        fs.int4_linear(x, w.to("cpu"))
    with pytest.raises(TypeError):
        fs.int4_linear(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        fs.int4_linear(x, w, out=torch.empty(2, 65, device=_dev()))
    with pytest.raises(ValueError):
        fs.int4_linear(x, w, out=torch.empty(64, 2, device=_dev()).T)
    with pytest.raises(ValueError):
        fs.int4_linear(x, w, out=torch.empty(2, 64, device=_dev()), out_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="backward"):
        fs.int4_linear(x.clone().requires_grad_(), w)
    with torch.no_grad():
        fs.int4_linear(x.clone().requires_grad_(), w)


_STATUS = """
import torch
import flashsampling_b200 as fs
from flashsampling_b200 import _lib, core
dev = torch.device("cuda", 0)
g = torch.Generator().manual_seed(0)
cpu = fs.Int4Weight.from_rows(torch.randint(0, 16, (300, 256), generator=g, dtype=torch.uint8), torch.full((300, 2), 0.01).bfloat16())
x = torch.randn(20, 256, generator=g).bfloat16().to(dev)
dense = torch.randn(512, 256, generator=g).bfloat16().to(dev)
qweight, scales = cpu.qweight.to(dev), cpu.scales.to(dev)
junk = [torch.full((1 << 20,), -1, dtype=torch.int32, device=dev) for _ in range(4)]
del junk
torch.cuda.synchronize()

# a weight of a capture, before anything made the status word: no call that needs it, and no word in the graph
early = torch.cuda.CUDAGraph()
with torch.cuda.graph(early):
    w = fs.Int4Weight(qweight, scales, None, 300, 256)
    few = fs.int4_linear(x[:3], w)
    try:
        fs.int4_linear(x, w)
        raise SystemExit("a product without a status word")
    except RuntimeError as e:
        assert "status word" in str(e)
    ids = fs.fused_mm_sample(dense, x, 1, None, 0, greedy_sampling=True)
assert not core._status
fs.check_status()
early.replay()
torch.cuda.synchronize()
assert torch.equal(ids[:, 0], (x.double() @ dense.double().T).argmax(1))

w = cpu.to(dev)
assert torch.equal(few, fs.int4_linear(x[:3], w))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = fs.int4_linear(x, w)
fs.check_status()  # nothing has run yet
core._status[0].fill_(_lib.ERR_TIMEOUT)  # as an earlier call's time-out
graph.replay()
try:
    fs.check_status()
    raise SystemExit("the replay cleared the word")
except _lib.FmmsError:
    pass
fs.check_status()
assert torch.equal(y, fs.int4_linear(x, w))
print("status kept")
"""


def test_status_word_of_a_process_whose_first_calls_are_captured(fs):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", _STATUS], cwd=root, capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and "status kept" in done.stdout, done.stdout[-500:] + done.stderr[-2000:]


@pytest.mark.parametrize("batch", [1, 6, 20])
def test_out_over_x_is_refused(fs, batch):
    w = _weight(fs, 256, 256, 64, False)
    x = _x(batch, 256, torch.bfloat16)
    want = fs.int4_linear(x, w)
    buf = torch.zeros(batch, 600, dtype=torch.bfloat16, device=_dev())
    buf[:, :256] = x
    for out in (buf[:, :256], buf[:, 128:384], buf[:, 255:511]):
        with pytest.raises(ValueError, match="share memory"):
            fs.int4_linear(buf[:, :256], w, out=out)
    fs.int4_linear(buf[:, :256], w, out=buf[:, 256:512])  # side by side
    assert torch.equal(buf[:, 256:512], want) and torch.equal(buf[:, :256], x)
