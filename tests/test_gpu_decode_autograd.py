"""The operators around a decode step beside autograd: derivatives are refused, writes into a caller's tensors are seen."""

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fs():
    import flashsampling_b200 as fs
    from flashsampling_b200 import build

    build.build_library()
    return fs


def _weight(fs, rows=48, cols=64):
    q = torch.randint(0, 16, (rows, cols), generator=torch.Generator().manual_seed(0), dtype=torch.uint8)
    return fs.Int4Weight.from_rows(q, torch.full((rows, cols // 32), 0.1).bfloat16()).to("cuda:0")


@pytest.mark.parametrize("batch", [2, 12])
def test_tangents_are_refused(fs, batch):
    w = _weight(fs)
    x = torch.randn(batch, 64, device="cuda:0").bfloat16()
    logits, scores, parents = torch.randn(1, 4, 50, device="cuda:0"), torch.zeros(1, 4, device="cuda:0"), torch.zeros(1, 4, dtype=torch.int64, device="cuda:0")
    out = torch.empty(batch, 48, device="cuda:0")
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: fs.int4_linear(dual(x), w), lambda: fs.int4_linear(x, w, out=dual(out)), lambda: fs.beam_search_step(dual(logits), scores),
                     lambda: fs.beam_search_step(logits, dual(scores)), lambda: fs.reorder_beams(dual(logits[0]), parents)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        fs.int4_linear(x, w, out=out)  # nothing carries a tangent
        fs.reorder_beams(logits[0], fs.beam_search_step(logits, scores).parents)


@pytest.mark.parametrize("batch", [2, 12])
def test_writes_raise_the_version(fs, batch):
    w = _weight(fs)
    x = torch.randn(batch, 64, device="cuda:0").bfloat16()
    out = torch.empty(batch, 48, device="cuda:0")
    before = out._version
    fs.int4_linear(x, w, out=out)
    assert out._version > before
    parents = torch.tensor([[1, 0, 3, 2]], device="cuda:0")
    states = [torch.randn(4, 8, device="cuda:0") for _ in range(3)]
    losses = [(s * torch.ones_like(s).requires_grad_()).sum() for s in (*states, out)]
    fs.reorder_beams(states, parents)
    with torch.no_grad():
        fs.int4_linear(x[:1], w, out=out[:1])
    for loss in losses:  # each has saved a tensor that is another one now
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()


def test_tensors_of_inference_mode_have_no_version(fs):
    with torch.inference_mode():
        w = _weight(fs)
        x = torch.randn(3, 64, device="cuda:0").bfloat16()
        state = torch.arange(8, device="cuda:0").view(4, 2)
        out = fs.int4_linear(x, w, out=torch.empty(3, 48, device="cuda:0"))
        fs.reorder_beams(state, torch.tensor([[1, 0, 3, 2]], device="cuda:0"))
    assert torch.equal(out, fs.int4_linear(x, w, out_dtype=torch.float32))
    assert state.tolist() == [[2, 3], [0, 1], [6, 7], [4, 5]]
