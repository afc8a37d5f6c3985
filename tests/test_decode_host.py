"""CPU tests of the operators around a decode step: the 4-bit layout and quantiser, the argument checks of the entry
points and of the C functions (all before any CUDA call), and the description of states for the reordering."""

import ctypes

import pytest
import torch

import flashsampling_b200 as fs
from flashsampling_b200 import _lib, beam
from flashsampling_b200.quant import quantize_groups_int4


def _codes(rows, cols, group, zeros, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 16, (rows, cols), generator=g, dtype=torch.uint8)
    s = (torch.rand(rows, cols // group, generator=g) + 0.5).to(torch.bfloat16)
    z = torch.randint(0, 16, (rows, cols // group), generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


@pytest.mark.parametrize("rows,cols,group,zeros", [(1, 32, 32, False), (16, 64, 64, True), (17, 96, 32, True), (40, 256, 256, False), (9, 768, 768, True), (33, 384, 128, True)])
def test_layout_follows_its_description(rows, cols, group, zeros):
    q, s, z = _codes(rows, cols, group, zeros)
    w = fs.Int4Weight.from_rows(q, s, z)
    assert w.shape == (rows, cols) and w.group_size == group
    flat = w.qweight
    for r in range(rows):
        for c in range(0, cols, 7):
            k = c % 16
            byte = (r % 8) * 64 + (k % 8 // 2) * 16 + (c % 64 // 16) * 4 + (k % 2) * 2 + k // 8
            assert int(flat[r // 16, c // 64, byte]) >> (4 * (r % 16 // 8)) & 15 == int(q[r, c])
            assert w.scales[r // 16, c // group, r % 8, r % 16 // 8] == s[r, c // group]
            if zeros:
                assert w.zeros[r // 16, c // group, r % 8, r % 16 // 8] == z[r, c // group]
    assert torch.equal(w.codes(), q)
    zero = 8 if z is None else z.double().repeat_interleave(group, 1)
    assert torch.equal(w.dequantize(torch.float64), (q.double() - zero) * s.double().repeat_interleave(group, 1))


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantiser_rounds_to_the_nearest_code(symmetric, dtype):
    w = (torch.randn(50, 256, generator=torch.Generator().manual_seed(1)) * 0.05).to(dtype)
    w[3] = 0
    w[4, :128] = 0.01  # one-sided group
    q, s, z = quantize_groups_int4(w, 128, symmetric)
    assert s.dtype == (dtype if dtype != torch.float32 else torch.bfloat16) and (z is None) == symmetric
    back = fs.Int4Weight.from_rows(q, s, z).dequantize(torch.float64)
    # half a step, plus what the rounding of the scale (eps / 2 relative, over up to 15 steps) and of the zero point
    # (half a step) can push beyond the last code
    step = s.double().repeat_interleave(128, 1)
    slack = 15 * torch.finfo(s.dtype).eps / 2 + (0 if symmetric else 0.5)
    assert bool(((back - w.double()).abs() <= step * (0.5 + slack) + 1e-12).all())
    assert bool((back[3] == 0).all())
    direct = fs.Int4Weight.quantize(w, 128, symmetric)
    assert torch.equal(direct.codes(), q)


def test_quantiser_refuses():
    w = torch.randn(4, 96)
    for bad in (dict(group_size=48), dict(group_size=64), dict(group_size=512), dict(group_size=96), dict(group_size=0), dict(group_size=-32)):
        with pytest.raises(ValueError):
            quantize_groups_int4(w, **bad)
    with pytest.raises(TypeError):
        quantize_groups_int4(w, 32, scale_dtype=torch.float32)
    with pytest.raises(ValueError):
        quantize_groups_int4(w[0], 32)
    with pytest.raises(ValueError):
        quantize_groups_int4(w.to(torch.int32), 32)


def test_int4_weight_refuses_other_layouts():
    q, s, z = _codes(20, 128, 64, True)
    w = fs.Int4Weight.from_rows(q, s, z)
    ok = (w.qweight, w.scales, w.zeros)
    with pytest.raises(ValueError):
        fs.Int4Weight(*ok, rows=0, cols=128)
    with pytest.raises(ValueError):
        fs.Int4Weight(*ok, rows=40, cols=128)  # another number of tiles
    with pytest.raises(ValueError):
        fs.Int4Weight(*ok, rows=20, cols=256)
    with pytest.raises(ValueError):
        fs.Int4Weight(w.qweight.to(torch.int8), w.scales, w.zeros, 20, 128)
    with pytest.raises(TypeError):
        fs.Int4Weight(w.qweight, w.scales.float(), w.zeros, 20, 128)
    with pytest.raises(ValueError):
        fs.Int4Weight(w.qweight, w.scales[:, :1].expand(-1, 3, -1, -1).contiguous(), None, 20, 128)  # 128 columns in 3 groups
    with pytest.raises(ValueError):
        fs.Int4Weight(w.qweight, w.scales, w.zeros.float(), 20, 128)
    with pytest.raises(ValueError):
        fs.Int4Weight(w.qweight, w.scales.transpose(2, 3), w.zeros, 20, 128)
    odd = torch.empty(w.qweight.numel() + 1, dtype=torch.uint8)[1:].view(w.qweight.shape)
    with pytest.raises(ValueError):
        fs.Int4Weight(odd, w.scales, w.zeros, 20, 128)  # not on a 16-byte boundary
    with pytest.raises(ValueError):
        fs.Int4Weight.from_rows(q, s[:10], None)
    with pytest.raises(ValueError):
        fs.Int4Weight.from_rows(q, s, z[:, :1])
    with pytest.raises(TypeError):
        fs.int4_linear(torch.zeros(1, 128, dtype=torch.bfloat16), w.dequantize())
    with pytest.raises(RuntimeError, match="CUDA"):
        fs.int4_linear(torch.zeros(1, 128, dtype=torch.bfloat16), w)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        fs.beam_search_step(torch.zeros(2, 3, 5), torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="CUDA"):
        fs.reorder_beams(torch.zeros(6, 5), torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):
        fs.BeamSearch(torch.zeros(8, 8, dtype=torch.bfloat16), 1, 2, 3)


def test_c_entry_points_check_their_arguments(lib):
    p = 4096  # never dereferenced
    ok = [p, 0, 64, p, p, 0, None, 100, 64, 64, 2, p, 2, 100, None, 0, None, None]

    def int4(**kw):
        names = "x x_dtype x_stride q s s_dtype z V D group B out out_dtype out_stride ws wsb status stream".split()
        return lib.fmms_int4_linear(*[kw.get(n, v) for n, v in zip(names, ok)])

    for kw in (dict(x=None), dict(q=None), dict(s=None), dict(out=None), dict(V=0), dict(D=0), dict(B=0), dict(B=-1),
               dict(x_dtype=2), dict(x_dtype=-1), dict(s_dtype=2), dict(out_dtype=3), dict(x_stride=63), dict(out_stride=99)):
        assert int4(**kw) == _lib.ERR_BAD_ARG, kw
    for kw in (dict(group=48), dict(group=128), dict(group=0), dict(group=-32), dict(group=16), dict(q=p + 8), dict(s=p + 2), dict(z=p + 4)):
        assert int4(**kw) == _lib.ERR_UNSUPPORTED, kw

    n = ctypes.c_size_t()
    assert lib.fmms_query_int4_workspace(151936, 4096, 128, 1, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.fmms_query_int4_workspace(128256, 8192, 128, 16, ctypes.byref(n)) == 0 and n.value >= 8192 * 16 * 2
    assert int4(D=8192, x_stride=8192, B=16, group=128) == _lib.ERR_WORKSPACE
    assert int4(D=8192, x_stride=8192, B=16, group=128, ws=p, wsb=64) == _lib.ERR_WORKSPACE
    assert lib.fmms_query_int4_workspace(100, 64, 128, 1, ctypes.byref(n)) == _lib.ERR_UNSUPPORTED
    assert lib.fmms_query_int4_workspace(100, 64, 64, 1, None) == _lib.ERR_BAD_ARG
    assert lib.fmms_query_beam_workspace(2, 4, 1000, 8, 0, ctypes.byref(n)) == 0 and n.value >= 8 * 8 * 8
    assert lib.fmms_query_beam_workspace(2, 4, 1000, 8, 3, ctypes.byref(n)) == _lib.ERR_BAD_ARG
    assert lib.fmms_query_beam_workspace(2, 4, 1000, 65, 0, ctypes.byref(n)) == _lib.ERR_UNSUPPORTED
    assert lib.fmms_query_beam_workspace(2, 4, 1000, 8, 0, None) == _lib.ERR_BAD_ARG
    beam_ok = [p, 0, 4000, 1000, p, None, 0, 2, 4, 1000, 8, p, p, p, p, 1 << 20, None]

    def step(**kw):
        names = "x dtype sr sk scores done pad R K V N os ot op ws wsb stream".split()
        return lib.fmms_beam_step(*[kw.get(m, v) for m, v in zip(names, beam_ok)])

    for kw in (dict(x=None), dict(scores=None), dict(os=None), dict(ot=None), dict(op=None), dict(R=0), dict(K=0), dict(V=0),
               dict(N=0), dict(dtype=3), dict(pad=-1), dict(pad=1000), dict(V=1, N=5), dict(x=p + 1), dict(x=p + 2, dtype=2)):
        assert step(**kw) == _lib.ERR_BAD_ARG, kw
    for kw in (dict(N=65), dict(K=65), dict(K=64, V=1 << 26), dict(R=1 << 16, K=1)):
        assert step(**kw) == _lib.ERR_UNSUPPORTED, kw
    for kw in (dict(ws=None), dict(ws=p + 8), dict(wsb=16)):
        assert step(**kw) == _lib.ERR_WORKSPACE, kw

    st = (_lib.FmmsBeamState * 1)()

    def reorder(**kw):
        d = dict(data=p, beam_stride=64, outer=(1, 1), seg_bytes=64, step_bytes=0, states=st, n=1, parents=p, pb=8, R=2, K=4)
        d.update(kw)
        st[0].data, st[0].beam_stride, st[0].seg_bytes, st[0].step_bytes = d["data"], d["beam_stride"], d["seg_bytes"], d["step_bytes"]
        st[0].outer[0], st[0].outer[1] = d["outer"]
        return lib.fmms_reorder_beams(d["states"], d["n"], d["parents"], d["pb"], d["R"], d["K"], None, None)

    for kw in (dict(states=None), dict(n=0), dict(parents=None), dict(pb=2), dict(R=0), dict(K=0), dict(data=None),
               dict(outer=(0, 1)), dict(outer=(1, -1)), dict(seg_bytes=0), dict(step_bytes=-1), dict(step_bytes=48)):
        assert reorder(**kw) == _lib.ERR_BAD_ARG, kw
    assert reorder(K=65) == _lib.ERR_UNSUPPORTED


def _moved(state, desc, R, K, parents, lengths):
    """What the kernel's addressing does with a described state, on the bytes of a CPU tensor's storage."""
    base = state.data_ptr()
    store = state.untyped_storage()
    raw = torch.empty(0, dtype=torch.uint8).set_(store)
    before = raw.clone()
    off0 = base - store.data_ptr()
    for o0 in range(desc.outer[0]):
        for o1 in range(desc.outer[1]):
            for r in range(R):
                live = desc.seg_bytes
                if lengths is not None and desc.step_bytes:
                    live = min(live, max(0, int(lengths[r])) * desc.step_bytes)
                seg = off0 + o0 * desc.outer_stride[0] + o1 * desc.outer_stride[1] + r * K * desc.beam_stride
                for j in range(K):
                    src, dst = seg + int(parents[r, j]) * desc.beam_stride, seg + j * desc.beam_stride
                    raw[dst:dst + live] = before[src:src + live]


@pytest.mark.parametrize("shape,dim,length_dim,perm", [
    ((6,), 0, None, None),
    ((6, 5), 0, 1, None),
    ((2, 6, 3, 4, 5), 1, 3, None),
    ((2, 6, 4, 3, 5), 1, 2, None),
    ((2, 2, 6, 3, 4), 2, 4, None),
    ((6, 3, 4, 5), 0, 2, (2, 0, 1, 3)),  # beams not outermost in memory
    ((6, 1, 4), 0, None, None),
    ((3, 6), 1, None, None),
])
def test_description_of_states(shape, dim, length_dim, perm):
    R, K = 2, 3
    g = torch.Generator().manual_seed(3)
    if perm is None:
        state = torch.randn(shape, generator=g)
    else:
        state = torch.randn([shape[i] for i in perm], generator=g).permute([perm.index(i) for i in range(len(perm))])
        assert state.shape == shape
        length_dim = None  # positions are not contiguous in this one
    parents = torch.tensor([[2, 0, 2], [1, 1, 0]])
    for lengths in ([None] if length_dim is None else [None, torch.tensor([1, 3], dtype=torch.int32)]):
        s = state.clone(memory_format=torch.preserve_format)
        assert s.stride() == state.stride()
        want = s.clone()
        for r in range(R):
            for j in range(K):
                src = state.select(dim, r * K + int(parents[r, j]))
                dst = want.select(dim, r * K + j)
                if lengths is None:
                    dst.copy_(src)
                else:
                    dst.narrow(length_dim - 1, 0, int(lengths[r])).copy_(src.narrow(length_dim - 1, 0, int(lengths[r])))
        desc = _lib.FmmsBeamState()
        beam._describe(s, dim, length_dim if lengths is not None else None, R, K, desc, lengths is not None)
        _moved(s, desc, R, K, parents, lengths)
        assert torch.equal(s, want)


def test_description_refuses():
    desc = _lib.FmmsBeamState()
    with pytest.raises(ValueError):  # another number of beams
        beam._describe(torch.zeros(5, 4), 0, None, 2, 3, desc, False)
    with pytest.raises(ValueError):  # shared memory
        beam._describe(torch.zeros(1, 4).expand(6, 4), 0, None, 2, 3, desc, False)
    with pytest.raises(ValueError):  # windows that overlap
        beam._describe(torch.zeros(20).unfold(0, 5, 3), 0, None, 2, 3, desc, False)
    with pytest.raises(ValueError):  # positions that are not contiguous
        beam._describe(torch.zeros(6, 4, 8)[..., ::2], 0, 1, 2, 3, desc, True)
    with pytest.raises(ValueError):  # three uneven dimensions around the beams
        beam._describe(torch.zeros(4, 3, 6, 4, 5)[::2, ::2, :, ::2], 2, None, 2, 3, desc, False)


def test_a_weight_keeps_its_tensors():
    """Calls pass on the addresses that the weight was made with: no attribute may change behind them."""
    import pickle

    q, s, z = _codes(20, 128, 64, True)
    w = fs.Int4Weight.from_rows(q, s, z)
    for name in ("qweight", "scales", "zeros", "rows", "_args"):
        with pytest.raises(AttributeError):
            setattr(w, name, None)
    again = pickle.loads(pickle.dumps(w))
    assert again.shape == w.shape and torch.equal(again.dequantize(), w.dequantize())


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantiser_refuses_what_a_scale_cannot_hold(symmetric):
    """A scale of infinity would make every weight of its group NaN."""
    for value, dtype in ((6e5, torch.float16), (float("inf"), torch.bfloat16), (float("nan"), torch.bfloat16), (-float("inf"), torch.float16)):
        w = torch.zeros(3, 64)
        w[1, 40] = value
        if not symmetric:
            w[1, 41] = -value
        with pytest.raises(ValueError, match="finite"):
            quantize_groups_int4(w, 32, symmetric, dtype)
        with pytest.raises(ValueError, match="finite"):
            fs.Int4Weight.quantize(w, 32, symmetric, dtype)
    w = torch.full((2, 32), 4e5)  # the largest scales of fp16 are scales
    w[1] = -4e5
    back = fs.Int4Weight.from_rows(*quantize_groups_int4(w, 32, symmetric, torch.float16)).dequantize()
    assert bool(((back - w).abs() <= 4e5 * (0.5 / 7 + 2.0**-10)).all())


def test_dynamic_shared_memory_has_one_alignment_per_name():
    """Kernels of a translation unit that declare the same array with different alignments get one of them."""
    import re

    from flashsampling_b200 import build

    def unit(path, seen):
        if path in seen or not path.exists():
            return ""
        seen.add(path)
        text = path.read_text()
        return text + "".join(unit((path.parent / name).resolve(), seen) for name in re.findall(r'#include "([^"]+)"', text))

    for source in build.SOURCES:
        found = {}
        for align, name in re.findall(r"extern __shared__ (?:__align__\((\d+)\) )?[\w ]+? (\w+)\[\]", unit(source.resolve(), set())):
            found.setdefault(name, set()).add(align)
        assert found and all(len(aligns) == 1 for aligns in found.values()), (source.name, found)


@pytest.mark.parametrize("name", ["qweight", "scales", "zeros"])
def test_a_weight_whose_tensors_moved_is_refused(name):
    for move in (lambda t: setattr(t, "data", t.clone()), lambda t: t.resize_(64, *t.shape[1:]), lambda t: t.untyped_storage().resize_(0)):
        w = fs.Int4Weight.from_rows(*_codes(20, 128, 64, True))
        assert w._call_args() == (w.qweight.data_ptr(), w.scales.data_ptr(), _lib.BF16, w.zeros.data_ptr(), 20, 128, 64)
        getattr(w, name).fill_(1)  # contents may change
        assert w._call_args() is w._args
        old = getattr(w, name).data  # keeps the memory, so that no other tensor gets its address
        move(getattr(w, name))
        if getattr(w, name).data_ptr() != w._args[("qweight", "scales", "", "zeros").index(name)]:
            with pytest.raises(RuntimeError, match="make a new Int4Weight"):
                w._call_args()
        else:
            raise AssertionError("the tensor has not moved")
        del old
    symmetric = fs.Int4Weight.from_rows(*_codes(20, 128, 64, False))
    assert symmetric._call_args()[3] is None


def test_c_entry_points_refuse_pointers_off_their_types(lib):
    """An element that does not lie on a multiple of its size would be a misaligned access on the GPU."""
    p = 4096  # never dereferenced

    def int4(x=p, out=p, out_dtype=0, status=None, batch=2):
        return lib.fmms_int4_linear(x, 0, 64, p, p, 0, None, 100, 64, 64, batch, out, out_dtype, 100, p, 1 << 30, status, None)

    for batch in (2, 20):
        for kw in (dict(x=p + 1), dict(out=p + 1), dict(out=p + 2, out_dtype=2), dict(out=p + 1, out_dtype=1), dict(status=p + 2)):
            assert int4(batch=batch, **kw) == _lib.ERR_BAD_ARG, kw

    def step(scores=p, os=p, ot=p, op=p):
        return lib.fmms_beam_step(p, 0, 4000, 1000, scores, None, 0, 2, 4, 1000, 8, os, ot, op, p, 1 << 20, None)

    for kw in (dict(scores=p + 2), dict(os=p + 1), dict(ot=p + 4), dict(op=p + 4)):
        assert step(**kw) == _lib.ERR_BAD_ARG, kw

    st = (_lib.FmmsBeamState * 1)()
    st[0].data, st[0].beam_stride, st[0].seg_bytes, st[0].outer[0], st[0].outer[1] = p, 64, 64, 1, 1
    for parents, size, lengths in ((p + 4, 8, None), (p + 2, 4, None), (p, 8, p + 2)):
        assert lib.fmms_reorder_beams(st, 1, parents, size, 2, 4, lengths, None) == _lib.ERR_BAD_ARG


def test_rows_that_share_memory_are_found():
    from types import SimpleNamespace

    from flashsampling_b200.int4 import _rows_meet

    g = torch.Generator().manual_seed(0)

    def r(lo, hi):
        return int(torch.randint(lo, hi, (1,), generator=g))

    found = set()
    for _ in range(2000):
        buf = torch.zeros(400, dtype=torch.bfloat16)
        b, cols, rows = r(1, 5), r(1, 12), r(1, 12)
        sx = cols + r(0, 20)
        so = sx if r(0, 2) and sx >= rows else rows + r(0, 20)
        x = buf.as_strided((b, cols), (sx, 1), r(0, 150))
        out = buf.as_strided((b, rows), (so, 1), r(0, 150))
        marks = torch.zeros(400, dtype=torch.int32)
        marks.as_strided(x.shape, x.stride(), x.storage_offset()).add_(1)
        want = bool((marks.as_strided(out.shape, out.stride(), out.storage_offset()) > 0).any())
        got = _rows_meet(x, sx, out, so, b, SimpleNamespace(rows=rows, cols=cols))
        assert got or not want  # nothing shared is missed
        if b == 1 or (sx == so and want):
            assert got == want
        found.add((want, got))
    assert {(False, False), (True, True)} <= found
    # x and out side by side in one buffer, and x over itself
    buf = torch.zeros(6, 30, dtype=torch.bfloat16)
    side = SimpleNamespace(rows=14, cols=16)
    assert not _rows_meet(buf[:, :16], 30, buf[:, 16:], 30, 6, side) and not _rows_meet(buf[:, 14:], 30, buf[:, :14], 30, 6, side)
    assert _rows_meet(buf[:, :16], 30, buf[:, 15:29], 30, 6, side) and _rows_meet(buf[:, :16], 30, buf[:, :14], 30, 6, side)


@pytest.mark.parametrize("eos", [None, 3])
def test_best_before_the_first_step_is_empty(eos):
    search = fs.BeamSearch.__new__(fs.BeamSearch)  # its tensors without a GPU
    search.requests, search.beams, search.max_steps, search.eos_token, search.pad_token, search.steps = 2, 3, 5, eos, 0, 0
    search.tokens = torch.zeros(6, 5, dtype=torch.int64)
    search.scores = torch.tensor([[0.0, -torch.inf, -torch.inf]]).repeat(2, 1)
    search.finished = torch.zeros(2, 3, dtype=torch.bool)
    tokens, scores = search.best(length_penalty=1.0)
    assert tokens.shape == (2, 0) and scores.tolist() == [0.0, 0.0]


def test_description_refuses_what_its_fields_cannot_hold():
    """Two beams of one byte each behind 2^32 + 5 blocks: 32 bits would make five of them."""
    desc = _lib.FmmsBeamState()
    for blocks in ((1 << 32) + 5, 1 << 31):
        with pytest.raises(ValueError, match="2\\^31"):
            beam._describe(torch.empty(blocks, 2, dtype=torch.uint8, device="meta"), 1, None, 1, 2, desc, False)
    beam._describe(torch.empty((1 << 31) - 1, 2, dtype=torch.uint8, device="meta"), 1, None, 1, 2, desc, False)
    assert desc.outer[1] == (1 << 31) - 1


def test_c_entry_points_refuse_sizes_that_overflow(lib):
    """Products and rounded multiples of 32-bit sizes: a query divided by R * K = 2^32 = 0, plans got negative step counts,
    and a kernel's column index would have wrapped."""
    big, n = 0x7FFFFFFF, ctypes.c_size_t()
    for sizes in ((1 << 26, 64, 1000, 8), (big, 64, 1000, 8), (65536, 1, 1000, 8), (1, 64, 1 << 25, 8)):
        assert lib.fmms_query_beam_workspace(*sizes, 0, ctypes.byref(n)) == _lib.ERR_UNSUPPORTED, sizes
    assert lib.fmms_query_beam_workspace(65535, 1, 1000, 8, 0, ctypes.byref(n)) == 0

    def both(V, D, group, B):
        p = 4096  # never dereferenced
        query = lib.fmms_query_int4_workspace(V, D, group, B, ctypes.byref(n))
        call = lib.fmms_int4_linear(p, 0, D, p, p, 0, None, V, D, group, B, p, 0, max(V, 1), None, 0, None, None)
        assert (query == _lib.ERR_UNSUPPORTED) == (call == _lib.ERR_UNSUPPORTED)
        return query

    for sizes in ((big, 64, 64, 1), (big - 14, 64, 64, 16), (100, big - 127 + 96, 32, 16), (100, (1 << 30) + 128, 128, 16), (100, (1 << 30) + 128, 128, 1),
                  (100, 64, 64, big), (100, 64, 64, 65535 * 64 + 1), (100, 64, 32, 65535 * 32 + 1)):
        assert both(*sizes) == _lib.ERR_UNSUPPORTED, sizes
    for sizes in ((big - 15, 64, 64, 16), (100, 1 << 30, 128, 16), (100, 64, 64, 65535 * 64), (100, 64, 32, 65535 * 32)):
        assert both(*sizes) == 0, sizes
        assert 0 < n.value < 1 << 45


def test_sizes_beyond_the_c_entry_points_are_refused(monkeypatch):
    """ctypes passes a Python integer of more than 32 bits on without its upper half."""
    with pytest.raises(ValueError, match="2\\^31"):
        fs.Int4Weight(torch.empty(((1 << 32) + 16) // 16, 1, 512, dtype=torch.uint8, device="meta"),
                      torch.empty(((1 << 32) + 16) // 16, 1, 8, 2, dtype=torch.bfloat16, device="meta"), None, (1 << 32) + 16, 32)
    with pytest.raises(ValueError, match="2\\^31"):
        beam._check_beams((1 << 31) + 1, 2)
    with pytest.raises(ValueError, match="64 beams"):
        beam._check_beams(3, 65)
    beam._check_beams((1 << 25) - 1, 64)


def test_a_status_word_of_inference_mode_is_cleared(monkeypatch):
    """A serving process makes the word and the workspaces under inference_mode and may check outside of it."""
    from flashsampling_b200 import core

    with torch.inference_mode():
        word, workspace = torch.full((1,), _lib.ERR_TIMEOUT, dtype=torch.int32), torch.ones(8, dtype=torch.uint8)
    monkeypatch.setattr(core, "_status", {None: word})  # (as a CPU tensor's device has it)
    monkeypatch.setattr(core, "_all_workspaces", [workspace])
    with pytest.raises(_lib.FmmsError):
        fs.check_status()
    assert int(word) == 0 and not bool(workspace.any())
    fs.check_status()
