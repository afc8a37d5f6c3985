"""The beam step, the reordering of states, and a search that runs both, against plain 64-bit computations.

Tolerance of the scores.  exp by the special-function unit is within 2^-22 relative, a thread adds at most 32 of them
in fp32 (32 2^-24), everything else is fp64: the sum is within 36 2^-24 + 2^-22 < 2^-18.6 relative, its logarithm within
2.6e-6 absolute; the output adds half an fp32 step of the score.  Tokens and parents have to be equal wherever the order
is decided by more than twice that (two beams' totals; within a beam the order is that of the logits, exactly).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
LSE = 2.6e-6


@pytest.fixture(scope="module")
def fs():
    import flashsampling_b200 as fs
    from flashsampling_b200 import build

    build.build_library()
    return fs


def _dev():
    return torch.device("cuda", 0)


def _reference(logits, scores, n, finished=None, pad=0):
    """(scores, tokens, parents, gap to the nearest candidate of another beam), one request at a time."""
    logits, scores = logits.cpu().double(), scores.cpu().double()
    R, K, V = logits.shape
    out_s = torch.full((R, n), -math.inf, dtype=torch.float64)
    out_t = torch.full((R, n), -1, dtype=torch.int64)
    out_p = torch.arange(n).clamp_max(K - 1).repeat(R, 1)
    gap = torch.full((R, n), math.inf, dtype=torch.float64)
    for r in range(R):
        cand = []
        for k in range(K):
            if not math.isfinite(scores[r, k]):
                continue
            if finished is not None and bool(finished[r, k]):
                cand.append((float(scores[r, k]), k, pad))
                continue
            x = logits[r, k].clone()
            x[x.isnan()] = -math.inf
            if x.max() == math.inf or x.max() == -math.inf:
                continue
            order = x.sort(descending=True, stable=True)
            lse = torch.logsumexp(x, 0)
            for v, i in zip(order.values[:n + 1].tolist(), order.indices[:n + 1].tolist()):
                if v > -math.inf:
                    cand.append((float(scores[r, k] + (v - lse)), k, i))
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        for i, (s, k, t) in enumerate(cand[:n]):
            out_s[r, i], out_t[r, i], out_p[r, i] = s, t, k
            others = [abs(c[0] - s) for c in cand[max(0, i - 1):i + 2] if c[1] != k]
            gap[r, i] = min(others, default=math.inf)
    return out_s, out_t, out_p, gap


def _check(step, ref):
    s, t, p, gap = ref
    got = step.scores.cpu().double()
    none = s == -math.inf
    assert torch.equal(got == -math.inf, none)
    tol = LSE + s.abs() * 2.0**-24
    assert bool(((got - s).abs()[~none] <= tol[~none]).all()), float((got - s)[~none].abs().max())
    clear = gap > 2 * LSE
    assert bool(clear.float().mean() > 0.9)
    assert torch.equal(step.tokens.cpu()[clear], t[clear]) and torch.equal(step.parents.cpu()[clear], p[clear])


def _inputs(R, K, V, dtype, seed, spread=2.2):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, V, generator=g) * spread
    x += (torch.rand(R, K, V, generator=g) < 24 / V) * (6 + 5 * torch.rand(R, K, V, generator=g))
    scores = -(8 * torch.rand(R, K, generator=g)).cumsum(1)
    return x.to(dtype).to(_dev()), scores.to(_dev())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,K,V,N", [(1, 1, 1, 1), (1, 1, 50, 7), (2, 3, 5, 15), (1, 4, 32000, 8), (3, 5, 4097, 5),
                                     (2, 8, 8192, 16), (2, 4, 8193, 17), (5, 2, 40001, 64), (1, 64, 3000, 64), (9, 33, 700, 33)])
def test_against_64_bits(fs, R, K, V, N, dtype):
    logits, scores = _inputs(R, K, V, dtype, seed=V + N)
    _check(fs.beam_search_step(logits, scores, num_candidates=N), _reference(logits, scores, N))


def test_large_vocabulary(fs):
    logits, scores = _inputs(6, 4, 262208, torch.bfloat16, seed=5)
    _check(fs.beam_search_step(logits, scores, num_candidates=8), _reference(logits, scores, 8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masks(fs, dtype):
    R, K, V, N = 6, 4, 5000, 8
    logits, scores = _inputs(R, K, V, dtype, seed=2)
    low = torch.finfo(dtype).min
    logits[0, :, 100:] = -math.inf
    logits[0, 1] = -math.inf  # nothing left
    logits[0, 2, 1:] = -math.inf  # one token left
    logits[1, :, ::2] = low
    logits[1, 0] = low  # all alike at the lowest value: every token has probability 1 / V
    logits[2, :, 50:300] = math.nan
    logits[2, 3] = math.nan
    logits[3, 2, 17] = math.inf  # no distribution
    logits[4] = -math.inf  # no candidate at all
    logits[5, :, 3:] = -math.inf  # fewer candidates than asked for
    logits[5, 1:] = -math.inf
    scores[2, 0] = -math.inf
    scores[3, 0] = math.nan
    scores[3, 1] = math.inf
    step = fs.beam_search_step(logits, scores, num_candidates=N)
    _check(step, _reference(logits, scores, N))
    assert step.tokens[4].tolist() == [-1] * N and step.parents[4].tolist() == [0, 1, 2, 3, 3, 3, 3, 3]
    assert (step.tokens[5] >= 0).sum() == 3


def test_equal_logits_go_to_the_lowest_token(fs):
    R, K, V, N = 4, 3, 20000, 12
    logits = torch.zeros(R, K, V, device=_dev())
    logits[1] = torch.randint(0, 3, (K, V), generator=torch.Generator().manual_seed(1)).float().to(_dev())
    logits[2, :, 700:] = 5.0  # more equal ones than any list holds
    logits[3, :, ::2] = -0.0  # -0 and 0 are equal
    scores = torch.tensor([[0.0, -0.5, -1.0]], device=_dev()).repeat(R, 1)
    step = fs.beam_search_step(logits, scores, num_candidates=N)
    _check(step, _reference(logits, scores, N))
    for r, first in ((0, list(range(N))), (2, list(range(700, 700 + N))), (3, list(range(N)))):
        assert step.tokens[r].tolist() == first and step.parents[r].tolist() == [0] * N
    # equal beams: the lower one first, token by token
    same = fs.beam_search_step(logits[:1], torch.zeros(1, K, device=_dev()), num_candidates=N)
    assert same.tokens[0].tolist() == list(range(N)) and same.parents[0].tolist() == [0] * N
    rows = logits[1:2, :1].expand(1, K, V)
    twice = fs.beam_search_step(rows, torch.zeros(1, K, device=_dev()), num_candidates=N)
    top = logits[1, 0].sort(descending=True, stable=True).indices[:N].tolist()
    assert twice.tokens[0].tolist() == top and twice.parents[0].tolist() == [0] * N


def test_candidates_crowded_in_one_place(fs):
    """The largest logits side by side, so that one thread, one slice or one beam holds all of them."""
    for V, dtype in ((3000, torch.float32), (40000, torch.bfloat16)):
        logits, scores = _inputs(2, 4, V, dtype, seed=9)
        logits[0, 1, 1000:1064] = torch.arange(30, 30 + 64, device=_dev()).to(dtype)
        logits[1] = torch.linspace(-20, 20, V, device=_dev()).to(dtype)  # rising over the vocabulary
        _check(fs.beam_search_step(logits, scores, num_candidates=64), _reference(logits, scores, 64))


def test_many_candidates_of_many_slices(fs):
    """More entries reach the merge's bound than its list holds: 64 beams of the same few tokens and scores."""
    K, V, N = 64, 30000, 64
    row = torch.zeros(V)
    row[::300] = 4.0
    logits = row.expand(1, K, V).contiguous().to(_dev())
    step = fs.beam_search_step(logits, torch.zeros(1, K, device=_dev()), num_candidates=N)
    assert step.tokens[0].tolist() == [300 * i for i in range(64)] and step.parents[0].tolist() == [0] * 64


def test_finished_beams(fs):
    R, K, V, N = 5, 4, 6000, 8
    logits, scores = _inputs(R, K, V, torch.bfloat16, seed=4)
    finished = torch.zeros(R, K, dtype=torch.bool, device=_dev())
    finished[0, 1] = finished[1, 0] = True
    finished[2] = True
    finished[3, :3] = True
    logits[2] = math.nan  # not read
    scores[3, 0] = -math.inf  # finished without a score: nothing
    for f in (finished, finished.to(torch.uint8) * 3):
        step = fs.beam_search_step(logits, scores, num_candidates=N, finished=f, pad_token=77)
        _check(step, _reference(logits, scores, N, finished, 77))
    assert step.tokens[2].tolist() == [77] * 4 + [-1] * 4
    assert torch.equal(step.scores[2, :4], scores[2].sort(descending=True).values)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_anywhere(fs, dtype):
    R, K, V, N = 3, 4, 5003, 8
    wide, scores = _inputs(R, K, 5100, dtype, seed=6)
    ref = None
    for start in range(0, 9):  # every alignment of a row
        view = wide[..., start:start + V]
        _check(fs.beam_search_step(view, scores, num_candidates=N), _reference(view, scores, N))
    view = wide.transpose(0, 1)[..., :V]  # beams outermost
    _check(fs.beam_search_step(view.transpose(0, 1), scores, num_candidates=N), _reference(wide[..., :V], scores, N))
    flat = wide.view(R * K, -1)[:, :V]
    ref = _reference(wide[..., :V], scores, N)
    _check(fs.beam_search_step(flat, scores.t().contiguous().t(), num_candidates=N), ref)


def test_step_streams_and_graphs(fs):
    logits, scores = _inputs(4, 4, 30000, torch.bfloat16, seed=7)
    other, scores2 = _inputs(4, 4, 30000, torch.bfloat16, seed=8)
    want = [fs.beam_search_step(x, s, num_candidates=8) for x, s in ((logits, scores), (other, scores2))]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    graphs = []
    for x, s in ((logits, scores), (other, scores2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = fs.beam_search_step(x, s, num_candidates=8)
        graphs.append((g, y))
    for _ in range(20):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, y), e in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(y, e))


def test_step_refusals(fs):
    logits, scores = _inputs(2, 3, 100, torch.float32, seed=1)
    bad = [
        (dict(logits=logits.double()), TypeError), (dict(scores=scores.double()), ValueError), (dict(scores=scores[:1]), ValueError),
        (dict(logits=logits[0, 0]), ValueError), (dict(logits=logits.view(6, 100)[:5]), ValueError),
        (dict(logits=logits.transpose(1, 2).contiguous().transpose(1, 2)), ValueError),
        (dict(num_candidates=0), ValueError), (dict(num_candidates=65), ValueError), (dict(logits=logits[..., :2], num_candidates=7), ValueError),
        (dict(pad_token=100), ValueError), (dict(pad_token=-1), ValueError), (dict(finished=torch.zeros(2, 2, dtype=torch.bool, device=_dev())), ValueError),
        (dict(finished=torch.zeros(2, 3, device=_dev())), ValueError), (dict(finished=torch.zeros(2, 3, dtype=torch.bool)), ValueError),
        (dict(scores=scores.cpu()), RuntimeError), (dict(logits=logits[..., :0]), ValueError), (dict(logits=logits.clone().requires_grad_()), RuntimeError),
        (dict(logits=torch.zeros(1, 65, 4, device=_dev()), scores=torch.zeros(1, 65, device=_dev())), ValueError),
    ]
    for kw, err in bad:
        with pytest.raises(err):
            fs.beam_search_step(**{**dict(logits=logits, scores=scores), **kw})
    empty = fs.beam_search_step(logits[:0], scores[:0])
    assert empty.tokens.shape == (0, 3)


# ------------------------------------------------------------------------------------------- reordering
def _reordered(state, parents, dim, lengths=None, length_dim=None):
    R, K = parents.shape
    want = state.clone()
    for r in range(R):
        for j in range(K):
            par = int(parents[r, j])
            par = j if not 0 <= par < K else par
            src, dst = state.select(dim, r * K + par), want.select(dim, r * K + j)
            if lengths is not None:
                n = min(max(int(lengths[r]), 0), state.shape[length_dim])
                ld = length_dim - 1 if length_dim > dim else length_dim
                src, dst = src.narrow(ld, 0, n), dst.narrow(ld, 0, n)
            dst.copy_(src)
    return want


def _fill(shape, dtype, seed):
    g = torch.Generator(device=_dev()).manual_seed(seed)
    if dtype.is_floating_point:
        return torch.randn(shape, generator=g, device=_dev()).to(dtype)
    return torch.randint(-100, 100, shape, generator=g, device=_dev()).to(dtype)


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16, torch.float32, torch.int64])
@pytest.mark.parametrize("R,K,rest", [(1, 2, (1,)), (3, 4, (5,)), (2, 3, (7, 11)), (4, 8, (3, 64)), (2, 5, (1000, 9)), (1, 16, (33, 40)),
                                      (2, 30, (77,)), (1, 64, (640,)), (1, 7, (2, 3, 4000)), (3, 1, (10,))])
def test_reorder(fs, R, K, rest, dtype):
    parents = torch.randint(0, K, (R, K), generator=torch.Generator().manual_seed(K)).to(_dev())
    for dim, shape in ((0, (R * K, *rest)), (1, (6, R * K, *rest)), (2, (2, 3, R * K, *rest))):
        state = _fill(shape, dtype, seed=K)
        want = _reordered(state, parents, dim)
        assert fs.reorder_beams(state, parents, dim=dim, length_dim=dim + 1) is None  # no lengths: whole beams
        assert _same(state, want)


@pytest.mark.parametrize("layout", ["bhtd", "bthd"])
@pytest.mark.parametrize("width,steps", [(64, 300), (41, 77), (1, 5), (128, 1), (8, 4096)])
def test_reorder_live_positions_only(fs, layout, width, steps):
    R, K, L, H = 7, 4, 3, 2
    lengths = torch.tensor([0, 1, steps, steps // 2, steps + 9, -3, max(0, steps - 1)], dtype=torch.int32, device=_dev())
    parents = torch.randint(0, K, (R, K), generator=torch.Generator().manual_seed(steps)).to(_dev())
    shape = (L, R * K, H, steps, width) if layout == "bhtd" else (L, R * K, steps, H, width)
    ld = 3 if layout == "bhtd" else 2
    for dtype in (torch.bfloat16, torch.float32):
        for lens in (lengths, lengths.long()):
            state = _fill(shape, dtype, seed=width)
            want = _reordered(state, parents, 1, lengths, ld)
            fs.reorder_beams(state, parents, dim=1, lengths=lens, length_dim=ld)
            assert _same(state, want)
        state = _fill(shape, dtype, seed=width)
        want = _reordered(state, parents, 1, lengths, ld)
        fs.reorder_beams(state, parents.int(), dim=-4, lengths=lengths, length_dim=ld - 5)
        assert _same(state, want)


def test_reorder_parents_that_are_no_beams_and_cycles(fs):
    parents = torch.tensor([[1, 2, 3, 0], [0, 0, 0, 0], [-1, 4, 1, 1 << 40], [3, 2, 1, 0], [0, 1, 2, 3]], device=_dev())
    state = _fill((20, 1000), torch.float32, seed=1)
    want = _reordered(state, parents.cpu(), 0)
    fs.reorder_beams(state, parents)
    assert _same(state, want) and torch.equal(state[16:], want[16:])


def test_reorder_views_and_many_states(fs):
    R, K = 3, 4
    parents = torch.randint(0, K, (R, K), generator=torch.Generator().manual_seed(0)).to(_dev())
    cache = _fill((70, 2, R * K, 16, 24), torch.bfloat16, seed=2)  # layer, key or value
    want = _reordered(cache, parents, 2)
    keys, values = [c[0] for c in cache], [c[1] for c in cache]
    fs.reorder_beams(keys + values, parents)  # 140 tensors
    assert _same(cache, want)
    big = _fill((R * K, 40, 100), torch.float32, seed=3)
    keep = big.clone()
    view = big[:, 3:20, 1:38]  # rows of odd alignment inside a larger buffer
    want = _reordered(view.clone(), parents, 0)
    fs.reorder_beams(view, parents)
    assert _same(view, want)
    keep[:, 3:20, 1:38] = want
    assert _same(big, keep)  # nothing around the view has changed
    inner = _fill((50, 5, R * K), torch.int64, seed=4).permute(2, 1, 0)  # beams innermost in memory
    want = _reordered(inner, parents, 0)
    fs.reorder_beams(inner, parents)
    assert _same(inner, want)
    fs.reorder_beams([], parents)
    fs.reorder_beams(torch.empty(R * K, 0, device=_dev()), parents)


def test_reorder_many_requests(fs):
    R, K = 1500, 3  # more than one launch takes
    parents = torch.randint(0, K, (R, K), generator=torch.Generator().manual_seed(0)).to(_dev())
    lengths = torch.randint(0, 41, (R,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(_dev())
    state = _fill((R * K, 40, 6), torch.float32, seed=5)
    live = (torch.arange(40, device=_dev()) < lengths.repeat_interleave(K)[:, None])[..., None]
    rows = (torch.arange(R, device=_dev())[:, None] * K + parents).flatten()
    want = torch.where(live, state[rows], state)
    fs.reorder_beams(state, parents, lengths=lengths, length_dim=1)
    assert _same(state, want)


def test_reorder_beyond_32_bits(fs):
    """A cache of more than 2^32 bytes: the last beams' offsets do not fit 32 bits."""
    R, K, T, D = 1, 4, 9_000_000, 128
    state = torch.empty((R * K, T, D), dtype=torch.uint8, device=_dev())
    state.copy_(torch.arange(K, dtype=torch.uint8, device=_dev())[:, None, None])
    lengths = torch.tensor([T - 1], dtype=torch.int32, device=_dev())
    fs.reorder_beams(state, torch.tensor([[3, 0, 2, 1]], device=_dev()), lengths=lengths, length_dim=1)
    for j, par in enumerate([3, 0, 2, 1]):
        assert bool((state[j, :-1] == par).all()) and bool((state[j, -1] == j).all())


def test_reorder_refusals(fs):
    parents = torch.zeros(2, 3, dtype=torch.int64, device=_dev())
    s = torch.zeros(6, 4, 5, device=_dev())
    lengths = torch.zeros(2, dtype=torch.int32, device=_dev())
    bad = [
        (dict(parents=parents.float()), ValueError), (dict(parents=parents[0]), ValueError), (dict(states=s[:5]), ValueError),
        (dict(states=s[:1].expand(6, 4, 5)), ValueError), (dict(states=[s, s]), ValueError), (dict(states=s.cpu()), RuntimeError),
        (dict(parents=parents.cpu()), RuntimeError), (dict(dim=3), ValueError), (dict(dim=1), ValueError), (dict(lengths=lengths), ValueError),
        (dict(lengths=lengths, length_dim=0), ValueError), (dict(lengths=lengths[:1], length_dim=1), ValueError),
        (dict(lengths=lengths.float(), length_dim=1), ValueError), (dict(lengths=lengths, length_dim=1, states=s.transpose(1, 2)), ValueError),
        (dict(states=torch.zeros(6, 4, device=_dev(), requires_grad=True)), RuntimeError),
        (dict(states=torch.zeros(65, 4, device=_dev()), parents=torch.zeros(1, 65, dtype=torch.int64, device=_dev())), ValueError),
    ]
    for kw, err in bad:
        with pytest.raises(err):
            fs.reorder_beams(**{**dict(states=s, parents=parents), **kw})


# ------------------------------------------------------------------------------------------- a search
def _plain_search(step_logits, R, K, steps, eos, pad):
    """Beam search in 64 bits on the CPU; step_logits(prefixes [R][K] of token tuples) -> [R, K, V]."""
    beams = [[((), 0.0, False)] for _ in range(R)]
    for _ in range(steps):
        for r in range(R):
            cand = []
            for k, (toks, sc, fin) in enumerate(beams[r]):
                if fin:
                    cand.append((sc, k, pad, True))
                    continue
                lp = torch.log_softmax(step_logits(r, toks).double(), 0)
                cand += [(sc + float(lp[v]), k, v, v == eos) for v in range(len(lp))]
            cand.sort(key=lambda c: (-c[0], c[1], c[2]))
            beams[r] = [(beams[r][k][0] + (v,), s, f) for s, k, v, f in cand[:K]]
    return beams


@pytest.mark.parametrize("eos", [7, 38, 191])  # on the CPU: no beam, one beam, three beams finish
@pytest.mark.parametrize("kind", ["bf16", "int4", "fp8"])
def test_search_on_every_head(fs, kind, eos):
    """Heads, selection, history, finished beams and states together: a toy language model whose hidden state is an
    embedding of the last two tokens, kept as a per-beam state that the search reorders."""
    from flashsampling_b200.quant import dequantize_rows, quantize_rows_e4m3
    from oracle import fmms_oracle as O

    R, K, V, D, steps, pad = 3, 4, 200, 64, 6, 1
    g = torch.Generator().manual_seed(11)
    w = (torch.randn(V, D, generator=g) * 0.35).bfloat16()
    w[eos] += 0.05
    emb = (torch.randn(V, D, generator=g) * 0.7).bfloat16()
    start = torch.randn(R, D, generator=g).bfloat16()
    if kind == "bf16":
        head, wd = w.to(_dev()), w
        logits = lambda h: (wd.double() @ h.double())  # noqa: E731
    elif kind == "int4":
        head = fs.Int4Weight.quantize(w, 32, symmetric=False).to(_dev())
        wd = fs.Int4Weight.quantize(w, 32, symmetric=False).dequantize(torch.float64)
        logits = lambda h: wd @ h.double()  # noqa: E731
    else:
        q, sc = quantize_rows_e4m3(w)
        head = (q.to(_dev()), sc.to(_dev()))
        logits = lambda h: O.quantized_logits(q, sc, h[None])[0].double()  # noqa: E731

    def hidden(r, toks):  # bf16 sums in the order of the GPU loop below
        prev = start[r]
        for t in toks:
            prev = (0.5 * prev.float() + emb[t].float()).bfloat16()
        return prev

    want = _plain_search(lambda r, toks: logits(hidden(r, toks)), R, K, steps, eos, pad)
    search = fs.BeamSearch(head, R, K, steps, eos_token=eos, pad_token=pad)
    emb_d = emb.to(_dev())
    h = start.repeat_interleave(K, 0).to(_dev())
    state = h.clone()
    for _ in range(steps):
        out = search.step(h, state)
        h = (0.5 * state.float() + emb_d[out.tokens.view(-1)].float()).bfloat16()
        state.copy_(h)
    fs.check_status()
    got_t, got_s = search.tokens.view(R, K, steps).cpu(), search.scores.cpu()
    ended = 0
    for r in range(R):
        for k in range(K):
            toks, sc, fin = want[r][k]
            assert got_t[r, k].tolist() == list(toks)
            assert abs(float(got_s[r, k]) - sc) < 1e-3 * steps  # logits within 1e-4 of their scale on every head
            assert bool(search.finished[r, k]) == fin
            ended += fin
    assert ended == {7: 0, 38: 1, 191: 3}[eos]
    tokens, score = search.best(length_penalty=1.0)
    for r in range(R):
        ranked = [s / (toks.index(eos) + 1 if eos in toks else steps) for toks, s, _ in want[r]]
        k = max(range(K), key=lambda i: ranked[i])
        assert tokens[r].tolist() == list(want[r][k][0]) and abs(float(score[r]) - ranked[k]) < 1e-3 * steps
    assert search.done() == all(f for b in want for _, _, f in b)
    with pytest.raises(RuntimeError):
        search.step(h)


def test_search_step_in_a_graph(fs):
    """One decode step - 4-bit head, beam step, caches - captured once and replayed on new inputs."""
    R, K, V, D, T = 2, 4, 5000, 256, 64
    w = fs.Int4Weight.quantize((torch.randn(V, D, generator=torch.Generator().manual_seed(1)) * 0.2).bfloat16(), 64).to(_dev())
    h = torch.zeros(R * K, D, dtype=torch.bfloat16, device=_dev())
    cache = torch.zeros(2, R * K, 3, T, 16, dtype=torch.bfloat16, device=_dev())
    scores = torch.zeros(R, K, device=_dev())
    lengths = torch.tensor([10, 64], dtype=torch.int32, device=_dev())

    def step():
        out = fs.beam_search_step(fs.int4_linear(h, w, out_dtype=torch.float32), scores)
        fs.reorder_beams(cache, out.parents, dim=1, lengths=lengths, length_dim=3)
        return out

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        g = torch.Generator(device=_dev()).manual_seed(seed)
        h.copy_(torch.randn(R * K, D, generator=g, device=_dev()))
        scores.copy_(-torch.rand(R, K, generator=g, device=_dev()))
        fresh = torch.randn(cache.shape, generator=g, device=_dev()).bfloat16()
        cache.copy_(fresh)
        eager = step()
        after = cache.clone()
        assert _same(after, _reordered(fresh, eager.parents, 1, lengths, 3))
        cache.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)) and _same(cache, after)


def test_reorder_states_of_every_width_at_once(fs):
    """Columns of 1, 2, 4, 8 and 16 bytes in one call, more than one launch's worth of one width among them."""
    g = torch.Generator(device=_dev()).manual_seed(11)
    r, k = 5, 6
    parents = torch.randint(0, k, (r, k), generator=g, device=_dev())
    shapes = [((r * k, 7), torch.uint8), ((r * k, 9), torch.bfloat16), ((r * k, 333, 3), torch.float32), ((r * k, 1), torch.int64),
              ((r * k, 40, 64), torch.bfloat16)] + [((r * k, 16 + i), torch.bfloat16) for i in range(130)]
    states = [torch.randint(0, 100, s, generator=g, device=_dev()).to(t) for s, t in shapes]
    at = (torch.arange(r, device=_dev())[:, None] * k + parents).view(-1)
    want = [s[at] for s in states]
    fs.reorder_beams(states, parents)
    assert all(torch.equal(s, w) for s, w in zip(states, want))


def test_search_that_runs_out_of_tokens(fs):
    """A head whose logits are all NaN leaves no token: no beam goes on, and the search is done."""
    w = torch.full((64, 32), float("nan"), device=_dev(), dtype=torch.bfloat16)
    weight = fs.Int4Weight.from_rows(torch.zeros(64, 32, dtype=torch.uint8, device=_dev()), w[:, :1].contiguous())
    search = fs.BeamSearch(weight, 2, 3, 4, eos_token=5)
    assert not search.done()
    out = search.step(torch.ones(6, 32, device=_dev(), dtype=torch.bfloat16))
    assert bool((out.scores == -float("inf")).all()) and search.done()


_CAPTURED_FIRST = """
import torch
import flashsampling_b200 as fs
dev = torch.device("cuda", 0)
g = torch.Generator().manual_seed(0)
q = torch.randint(0, 16, (300, 256), generator=g, dtype=torch.uint8).to(dev)
w = fs.Int4Weight.from_rows(q, torch.full((300, 2), 0.01, device=dev).bfloat16())
h = torch.randn(4, 256, generator=g).bfloat16().to(dev)
many = torch.randn(20, 256, generator=g).bfloat16().to(dev)
scores = torch.zeros(1, 4, device=dev)
state = torch.arange(4 * 5, device=dev).view(4, 5)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    logits = fs.int4_linear(h, w, out_dtype=torch.float32)
    more = fs.int4_linear(many, w, out_dtype=torch.float32)
    step = fs.beam_search_step(logits, scores)
    fs.reorder_beams(state, step.parents)
graph.replay()
torch.cuda.synchronize()
eager = fs.beam_search_step(fs.int4_linear(h, w, out_dtype=torch.float32), scores)
assert torch.equal(eager.tokens, step.tokens) and torch.equal(eager.parents, step.parents) and torch.equal(eager.scores, step.scores)
assert torch.equal(more, fs.int4_linear(many, w, out_dtype=torch.float32))
assert torch.equal(state, torch.arange(4 * 5, device=dev).view(4, 5)[step.parents[0]])
fs.check_status()
print("captured first")
"""


def test_first_calls_of_a_process_inside_a_capture(fs):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", _CAPTURED_FIRST], cwd=root, capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and "captured first" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("kind", ["spread", "equal", "one beam", "dead", "falling"])
@pytest.mark.parametrize("K,V,N,dtype", [(10, 50000, 20, torch.float32), (12, 70001, 24, torch.bfloat16), (5, 120000, 64, torch.float16)])
def test_many_lists_to_join(fs, K, V, N, dtype, kind):
    """More entries than the join holds at a time: as a rule few of them matter; with equal logits all do."""
    R = 2
    logits, scores = _inputs(R, K, V, dtype, seed=K + N)
    finished = torch.zeros(R, K, dtype=torch.bool, device=_dev())
    if kind == "equal":
        logits = torch.ones_like(logits)
        scores = torch.zeros_like(scores)
    elif kind == "one beam":  # the others finished or without a score
        finished[:, 1:3] = True
        scores[:, 3:] = -math.inf
    elif kind == "dead":
        logits[0, 1:] = -math.inf
        logits[0, 0, N // 2:] = -math.inf  # fewer candidates than asked for
        finished[1, 0] = True
    elif kind == "falling":  # all of the best in the first lists
        logits = logits.sort(dim=-1, descending=True).values
    step = fs.beam_search_step(logits, scores, num_candidates=N, finished=finished, pad_token=3)
    ref = _reference(logits, scores, N, finished, 3)
    if kind == "equal":  # totals of different beams are equal: the lowest beam's first tokens
        assert step.parents.eq(0).all() and torch.equal(step.tokens.cpu(), torch.arange(N).repeat(R, 1))
    else:
        _check(step, ref)


@pytest.mark.parametrize("V", [600, 1000, 1500, 2047])
@pytest.mark.parametrize("N", [5, 24, 64])
def test_short_rows(fs, V, N):
    """Rows whose vectors do not fill the groups that a bound is taken from."""
    logits, scores = _inputs(3, 4, V, torch.bfloat16, seed=V + N)
    _check(fs.beam_search_step(logits, scores, num_candidates=N), _reference(logits, scores, N))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [7, 1501, 32003, 50257, 128257])
def test_equal_beams_that_lie_anywhere(fs, V, dtype):
    """Beams with the same logits and scores, each in a row of its own: an odd number of tokens puts every row elsewhere
    between two 16-byte boundaries, and equal totals come in the order of (beam, token) all the same."""
    R, K, N = 2, 8, 24
    row = _inputs(R, 1, V, dtype, seed=V)[0]
    wide = torch.full((R, K, V + 6), math.nan, dtype=dtype, device=_dev())  # NaN around the rows: no row reads beyond itself
    even = torch.zeros((R, K, V + 8 - V % 8), dtype=dtype, device=_dev())
    even[..., :V] = row
    for logits in (row.expand(R, K, V).contiguous(), even[..., :V], wide[..., 1:V + 1], wide[..., 4:V + 4]):
        logits.copy_(row.expand(R, K, V))
        step = fs.beam_search_step(logits, torch.full((R, K), -3.7, device=_dev()), num_candidates=N)
        for r in range(R):
            x = row[r, 0].tolist()
            top = sorted(range(V), key=lambda v: (-x[v], v))[:N]
            want = sorted(((k, v) for k in range(K) for v in top), key=lambda c: (-x[c[1]], c[0], c[1]))[:N]
            assert list(zip(step.parents[r].tolist(), step.tokens[r].tolist())) == want
        wide.fill_(math.nan)


def _lse_errors(fs, logits):
    """Errors of the log-sum-exps of rows [K, V]: a score that cancels the best token's log-probability leaves a total so
    near zero that the fp32 output shows them."""
    x = logits.cpu().double()
    lse, top = torch.logsumexp(x, 1), x.amax(1)
    scores = (lse - top).float()
    step = [fs.beam_search_step(logits[k].view(1, 1, -1), scores[k].view(1, 1).to(_dev()), num_candidates=1).scores for k in range(len(x))]
    return torch.cat(step).view(-1).cpu().double() - (scores.double() + (top - lse))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [40, 5000, 262208])
def test_log_sum_exp_within_what_is_claimed(fs, V, dtype):
    """Per exponential 2^-22 for the special-function unit and 2^-24 |x - max| for the rounding of the difference, whose
    mean over the softmax is at most ln V; 11 fp32 additions of 2^-24 (3 in a pass over two vectors, 8 passes); the rest
    is fp64: (4 + 11 + ln V) 2^-24 relative, which is the logarithm's absolute error (below 2e-6 for 2^18 tokens)."""
    g = torch.Generator().manual_seed(V)
    rows = [
        torch.randn(V, generator=g) * 2.2,  # a wide one
        torch.randn(V, generator=g) * 8,  # a peaked one
        torch.rand(V, generator=g) * 0.7,  # a flat one
        torch.where(torch.rand(V, generator=g) < 0.5, -0.3, 0.0),  # two values
        torch.randn(V, generator=g) * 2.2 - 30,  # log-probabilities
        torch.cat([torch.tensor([11.3, 11.1, 10.7]), torch.randn(V - 3, generator=g)]),  # three tokens with the mass
        torch.linspace(-20, 20, V),
    ]
    errors = _lse_errors(fs, torch.stack(rows).to(dtype).to(_dev()))
    assert bool((errors.abs() <= (15 + math.log(V)) * 2.0**-24).all()), errors


def test_exponentials_carry_the_rounding_of_their_arguments(fs):
    """Tokens d below the maximum, where d log2(e) rounds by half a step of fp32: 2^-20, with what fp32 cuts off log2(e)
    8e-7 of their share of the sum.  Carried along, what is left is the special-function unit's 2^-22: d is a bf16
    number, a thread's sum of 8 or 16 equal numbers in pairs is exact, and the maxima (one in 4096 tokens: every slice's
    reference) stand alone in their threads, whose other tokens (within 8 of a multiple of 1024) are masked."""
    V, log2e = 262208, 1.4426950408889634
    d = -torch.arange(11.125, 12, 0.0625)
    off = d.double() * log2e - (d * torch.tensor(log2e, dtype=torch.float32)).double()
    at = int(off.abs().argmax())
    x = torch.full((1, V), float(d[at]))
    x[:, torch.arange(V) % 1024 < 8] = -math.inf
    x[:, ::4096] = 0
    mass = int((x == d[at]).sum()) * math.exp(float(d[at]))
    share = mass / (mass + int((x == 0).sum()))
    tol = share * 2.0**-22 + 1e-9
    assert share * (float(off[at].abs()) * math.log(2) - 2.0**-22) > 2 * tol  # without it, errors are larger than this
    for dtype in (torch.bfloat16, torch.float32):
        assert abs(float(_lse_errors(fs, x.to(dtype).to(_dev()))[0])) <= tol


def test_sums_join_in_more_than_32_bits(fs):
    """Equal logits: exponentials and a thread's sums are exact, and 2^24 + 3 of them are more than fp32 can count.  A beam
    with one token fewer has probabilities that are larger by 6e-8, and comes first."""
    V, K = (1 << 24) + 3, 2
    logits = torch.zeros(K, V, dtype=torch.bfloat16, device=_dev())
    logits[1, 7] = -math.inf
    assert bool((_lse_errors(fs, logits).abs() <= 1e-10).all())
    step = fs.beam_search_step(logits[None], torch.full((1, K), -2.5, device=_dev()), num_candidates=5)
    assert step.parents[0].tolist() == [1] * 5 and step.tokens[0].tolist() == [0, 1, 2, 3, 4]
