"""Beam search next to sampling: the selection over beams and vocabulary, the reordering of per-beam states, and a
searcher that runs both behind any of the framework's heads.

``beam_search_step`` and ``reorder_beams`` are single calls on CUDA tensors (``csrc/fmms_beam.cuh``,
``csrc/fmms_reorder.cuh``), without synchronisation, so that a decode step can be captured in a CUDA graph.
``BeamSearch`` keeps the scores, the token histories and the finished beams of a batch of requests.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Sequence

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from .core import _refuse_gradients, _status_word
from .int4 import Int4Weight, int4_linear

__all__ = ["BeamStep", "beam_search_step", "reorder_beams", "BeamSearch"]

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}
_ws_bytes: dict[tuple, int] = {}


class BeamStep(NamedTuple):
    """The candidates of a step, best first: ``[requests, num_candidates]`` each."""

    scores: torch.Tensor  # fp32; -inf where there is no candidate
    tokens: torch.Tensor  # int64; -1 where there is no candidate
    parents: torch.Tensor  # int64, the beam 0..beams-1 that the candidate continues


def beam_search_step(
    logits: torch.Tensor,  # [requests, beams, vocab] or [requests * beams, vocab], bf16 / fp16 / fp32
    scores: torch.Tensor,  # [requests, beams] fp32: log-probability of every beam so far
    num_candidates: int | None = None,  # default: the number of beams
    finished: torch.Tensor | None = None,  # [requests, beams] bool or uint8
    pad_token: int = 0,
) -> BeamStep:
    """Of all continuations (beam ``k``, token ``v``) of every request the ``num_candidates`` with the largest
    ``scores[r, k] + log_softmax(logits[r, k])[v]``, best first; equal ones in the order of ``(k, v)``.

    NaN and ``-inf`` logits are tokens that may not follow.  A row with ``+inf``, or with nothing above ``-inf``, gives
    no candidate, nor does a beam whose score is not finite (a first step starts from scores ``[0, -inf, ...]``).  A
    finished beam goes on as it is: its one candidate is ``pad_token`` with its unchanged score.  Where fewer than
    ``num_candidates`` exist, the rest is score ``-inf``, token ``-1``, parent ``min(position, beams - 1)``.

    Exponentials and the sums of a thread are fp32, joined sums, logarithms and totals 64-bit: a log-softmax is within
    ``(15 + ln vocab) 2^-24`` (2e-6 for 2^18 tokens; measured 1e-7).  Candidates of two beams that lie closer together may
    come in either order, which may also change with the size of the batch; within a beam, and between beams of equal logits and
    scores, the order is exact.  Up to 64 beams and 64 candidates.  Rows may lie anywhere
    (``logits[..., :vocab]`` of a padded head needs no copy), their elements must be consecutive.  No gradients."""
    if not (logits.is_cuda and scores.is_cuda):
        raise RuntimeError("beam_search_step requires CUDA tensors (there is no CPU path)")
    if logits.dtype not in _DTYPES:
        raise TypeError("logits must be bfloat16, float16 or float32")
    if scores.ndim != 2 or scores.dtype is not torch.float32:
        raise ValueError("scores must be fp32 [requests, beams]")
    R, K = scores.shape
    dev = logits.device
    if logits.ndim == 3:
        if logits.shape[0] != R or logits.shape[1] != K:
            raise ValueError(f"logits must be [{R}, {K}, vocab], got {list(logits.shape)}")
        stride_r, stride_k = logits.stride(0), logits.stride(1)
    elif logits.ndim == 2:
        if logits.shape[0] != R * K:
            raise ValueError(f"logits must be [{R * K}, vocab], got {list(logits.shape)}")
        stride_k = logits.stride(0)
        stride_r = K * stride_k
    else:
        raise ValueError("logits must be [requests, beams, vocab] or [requests * beams, vocab]")
    V = logits.shape[-1]
    N = K if num_candidates is None else int(num_candidates)
    if scores.device != dev or (finished is not None and finished.device != dev):
        raise ValueError(f"scores and finished must be on the logits' device ({dev})")
    if K < 1 or V < 1 or not 1 <= N <= 64 or K > 64:
        raise ValueError("beam_search_step takes 1 to 64 beams, 1 to 64 candidates and at least one token")
    if N > K * V:
        raise ValueError(f"{N} candidates of {K} x {V} continuations")
    if K * V >= 1 << 31 or R * K > 65535:
        raise ValueError("beam_search_step takes beams * vocab < 2^31 and requests * beams <= 65535")
    if not 0 <= pad_token < V:
        raise ValueError(f"pad_token must be one of the {V} tokens")
    if V > 1 and logits.stride(-1) != 1:
        raise ValueError("the logits of a row must be consecutive")
    if logits.requires_grad or scores.requires_grad or forward_ad._current_level >= 0:
        _refuse_gradients("beam_search_step", logits, scores)
    if not scores.is_contiguous():
        scores = scores.contiguous()
    done = None
    if finished is not None:
        if finished.shape != (R, K) or finished.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"finished must be bool or uint8 [{R}, {K}]")
        finished = finished.contiguous()
        done = finished.data_ptr()
    step = BeamStep(
        # empty_strided: the allocation with the least host time
        torch.empty_strided((R, N), (N, 1), dtype=torch.float32, device=dev),
        torch.empty_strided((R, N), (N, 1), dtype=torch.int64, device=dev),
        torch.empty_strided((R, N), (N, 1), dtype=torch.int64, device=dev),
    )
    if R == 0:
        return step
    dt = _DTYPES[logits.dtype]
    key = (R, K, V, N, dt)
    nbytes = _ws_bytes.get(key)
    if nbytes is None:
        nbytes = _ws_bytes[key] = _lib.query_beam_workspace(*key)
    # from torch's allocator on every call: calls on several streams, or in several captured graphs, share nothing
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    index = dev.index
    args = (
        logits.data_ptr(), dt, stride_r, stride_k, scores.data_ptr(), done, int(pad_token), R, K, V, N,
        step.scores.data_ptr(), step.tokens.data_ptr(), step.parents.data_ptr(), ws.data_ptr(), nbytes,
        torch._C._cuda_getCurrentRawStream(index),
    )
    if torch._C._cuda_getDevice() == index:
        rc = _lib.load().fmms_beam_step(*args)
    else:
        with torch.cuda.device(dev):
            rc = _lib.load().fmms_beam_step(*args)
    if rc:
        raise _lib.FmmsError(rc, "fmms_beam_step")
    return step


def _merge_dims(dims: list[tuple[int, int]]) -> list[tuple[int, int]]:
    """(size, stride) pairs, outermost first, with neighbours joined where they are one even sequence."""
    out: list[tuple[int, int]] = []
    for size, stride in dims:
        if size == 1:
            continue
        if out and out[-1][1] == size * stride:
            out[-1] = (out[-1][0] * size, stride)
        else:
            out.append((size, stride))
    return out


def _describe(s: torch.Tensor, dim: int, length_dim: int | None, R: int, K: int, desc: "_lib.FmmsBeamState",
              lengths: bool) -> None:
    """Fill ``fmms_beam_state_t`` for one state: blocks around the beams, and one contiguous run per beam and block."""
    es = s.element_size()
    if s.shape[dim] != R * K:
        raise ValueError(f"a state has {s.shape[dim]} beams along dimension {dim}, parents is for {R} x {K}")
    sizes, strides = s.shape, s.stride()
    span = 1
    for st, n in sorted(zip(strides, sizes)):
        if n > 1:
            if st < span:
                raise ValueError("a state must not be an expanded or overlapping view: its elements would share memory")
            span += (n - 1) * st
    # the innermost dimensions that make one contiguous run; positions are its outermost dimension
    run, first = 1, s.ndim
    while first > dim + 1 and (sizes[first - 1] == 1 or strides[first - 1] == run):
        first -= 1
        run *= sizes[first]
        if lengths and first == length_dim:
            break
    step = 0
    if lengths:
        if first != length_dim:
            raise ValueError(f"the elements of a state from dimension {length_dim} (positions) on must be contiguous")
        step = run // sizes[length_dim] * es if sizes[length_dim] else 0
    blocks = _merge_dims([(sizes[i], strides[i]) for i in range(s.ndim) if i != dim and i < first])
    if len(blocks) > 2:
        raise ValueError("a state's dimensions around the beams must form at most two even sequences")
    while len(blocks) < 2:
        blocks.insert(0, (1, 0))
    if blocks[0][0] >= 1 << 31 or blocks[1][0] >= 1 << 31:
        raise ValueError("a state's dimensions around the beams must be below 2^31 blocks each")
    desc.data = s.data_ptr()
    desc.beam_stride = strides[dim] * es
    desc.outer_stride[0], desc.outer_stride[1] = blocks[0][1] * es, blocks[1][1] * es
    desc.outer[0], desc.outer[1] = blocks[0][0], blocks[1][0]
    desc.seg_bytes = run * es
    desc.step_bytes = step


def _check_beams(R: int, K: int) -> None:
    if K < 1 or K > 64:
        raise ValueError("reorder_beams takes 1 to 64 beams")
    if R * K >= 1 << 31:
        raise ValueError("reorder_beams takes requests * beams < 2^31")


def reorder_beams(
    states: torch.Tensor | Sequence[torch.Tensor],  # any type; dimension `dim` is [requests * beams]
    parents: torch.Tensor,  # [requests, beams] int64 or int32
    dim: int = 0,
    lengths: torch.Tensor | None = None,  # [requests] int32 or int64: positions in use
    length_dim: int | None = None,  # the states' dimension of positions, behind `dim`
) -> None:
    """Beam ``j`` of request ``r`` continues beam ``parents[r, j]``: in every state, in place,
    ``state[.., r * beams + j, ..] = state[.., r * beams + parents[r, j], ..]``, all beams at once.

    Without ``lengths`` whole beams move.  With ``lengths`` only the first ``lengths[r]`` positions along ``length_dim`` do;
    what lies behind them stays as it is (lengths beyond the dimension count as all of it).  A parent outside ``0..beams-1`` keeps the beam's own state.
    One launch for up to 64 tensors; a beam that keeps its own state costs no traffic.  Up to 64 beams.  States may
    be strided views as long as they do not overlap, themselves or one another."""
    states = [states] if isinstance(states, torch.Tensor) else list(states)
    if parents.ndim != 2 or parents.dtype not in (torch.int64, torch.int32):
        raise ValueError("parents must be int64 or int32 [requests, beams]")
    if not parents.is_cuda or not all(s.is_cuda for s in states):
        raise RuntimeError("reorder_beams requires CUDA tensors (there is no CPU path)")
    R, K = parents.shape
    _check_beams(R, K)
    dev = parents.device
    if lengths is not None and length_dim is None:
        raise ValueError("lengths needs length_dim, the states' dimension of positions")
    if lengths is not None:
        if lengths.shape != (R,) or lengths.dtype not in (torch.int32, torch.int64) or lengths.device != dev:
            raise ValueError(f"lengths must be int32 or int64 [{R}] on {dev}")
        if lengths.dtype is torch.int64:
            lengths = lengths.clamp(0, 0x7fffffff).to(torch.int32)
        lengths = lengths.contiguous()
    parents = parents.contiguous()
    descs = (_lib.FmmsBeamState * max(1, len(states)))()
    n, seen, dual = 0, set(), forward_ad._current_level >= 0
    for s in states:
        if s.device != dev:
            raise ValueError(f"a state is on {s.device}, parents on {dev}")
        if s.requires_grad or dual:
            _refuse_gradients("reorder_beams (in place)", s)
        if s.is_complex() or s.is_sparse or s.is_quantized:
            raise TypeError("states must be plain dense tensors")
        d = dim + s.ndim if dim < 0 else dim
        ld = None if lengths is None else (length_dim + s.ndim if length_dim < 0 else length_dim)
        if not 0 <= d < s.ndim or (ld is not None and not d < ld < s.ndim):
            raise ValueError(f"a state of {s.ndim} dimensions has no beams along {dim}, or no positions behind them along {length_dim}")
        _describe(s, d, ld, R, K, descs[n], lengths is not None)
        if s.numel() == 0:
            continue
        if s.data_ptr() in seen:
            raise ValueError("the same state twice: it would be reordered twice")
        seen.add(s.data_ptr())
        n += 1
    if n == 0 or R == 0 or K == 1:
        return
    index = dev.index
    args = (descs, n, parents.data_ptr(), parents.element_size(), R, K, lengths.data_ptr() if lengths is not None else None,
            torch._C._cuda_getCurrentRawStream(index))
    if torch._C._cuda_getDevice() == index:
        rc = _lib.load().fmms_reorder_beams(*args)
    else:
        with torch.cuda.device(dev):
            rc = _lib.load().fmms_reorder_beams(*args)
    if rc:
        raise _lib.FmmsError(rc, "fmms_reorder_beams")
    increment_version(states)  # as torch's own operations do: what autograd has saved of them is no longer there


class BeamSearch:
    """Beam search of ``requests`` sequences with ``beams`` hypotheses each behind one LM head.

    ``head`` is what the framework samples or multiplies with: a bf16 ``[vocab, hidden]`` weight, an
    ``Int4Weight``, or a pair ``(float8_e4m3fn weight, fp32 row scales)``.  ``step(hidden_states)`` takes the
    hidden states ``[requests * beams, hidden]`` of the current tokens, chooses every request's next beams, and reorders
    the token histories and the caller's per-beam ``states`` in place; ``tokens``, ``scores`` and ``finished`` hold
    the hypotheses, best first.  A beam that took ``eos_token`` is finished: it keeps its score, its tokens go on with
    ``pad_token``, and it competes with the others until ``done()``.  Nothing synchronises with the host except
    ``done()`` and ``best()``.
    """

    def __init__(self, head, requests: int, beams: int, max_steps: int, eos_token: int | None = None, pad_token: int = 0):
        self.head = head
        if isinstance(head, Int4Weight):
            dev = head.device
        elif isinstance(head, tuple):
            dev = head[0].device
        else:
            dev = head.device
        if dev.type != "cuda":
            raise RuntimeError("BeamSearch requires a head on a GPU (there is no CPU path)")
        if requests < 1 or max_steps < 1 or not 1 <= beams <= 64:
            raise ValueError("BeamSearch takes at least one request and one step, and 1 to 64 beams")
        _status_word(dev)  # here, for the first step may be inside a capture
        self.requests, self.beams, self.max_steps = requests, beams, max_steps
        self.eos_token, self.pad_token = eos_token, pad_token
        self.tokens = torch.full((requests * beams, max_steps), pad_token, dtype=torch.int64, device=dev)
        self.scores = torch.full((requests, beams), -math.inf, dtype=torch.float32, device=dev)
        self.scores[:, 0] = 0  # all beams of a request start alike: only the first may branch
        self.finished = torch.zeros((requests, beams), dtype=torch.bool, device=dev)
        self.steps = 0

    def logits(self, hidden_states: torch.Tensor) -> torch.Tensor:
        """``[requests * beams, vocab]`` fp32 logits of the head."""
        from .core import fused_mm_sample

        if isinstance(self.head, Int4Weight):
            return int4_linear(hidden_states, self.head, out_dtype=torch.float32)
        weight, scale = self.head if isinstance(self.head, tuple) else (self.head, None)
        return fused_mm_sample(weight, hidden_states, 1, None, 0, greedy_sampling=True, return_logits=True,
                               weight_scale=scale)[1]

    def step(self, hidden_states: torch.Tensor, states: torch.Tensor | Sequence[torch.Tensor] = (), dim: int = 0,
             lengths: torch.Tensor | None = None, length_dim: int | None = None) -> BeamStep:
        """One token for every beam.  ``states`` (with ``dim``, ``lengths``, ``length_dim`` as in ``reorder_beams``) are
        reordered along; the returned ``tokens`` are the next inputs of the beams."""
        if self.steps >= self.max_steps:
            raise RuntimeError(f"the search was made for {self.max_steps} steps")
        out = beam_search_step(self.logits(hidden_states), self.scores, finished=self.finished, pad_token=self.pad_token)
        if isinstance(states, torch.Tensor) or len(states):
            reorder_beams(states, out.parents, dim=dim, lengths=lengths, length_dim=length_dim)
        reorder_beams(self.tokens, out.parents)
        tokens = out.tokens.clamp_min(0)  # a beam without a continuation (score -inf) stays without one
        self.tokens[:, self.steps] = tokens.view(-1)
        self.scores.copy_(out.scores)
        finished = self.finished.gather(1, out.parents)
        if self.eos_token is not None:
            finished |= tokens == self.eos_token
        self.finished.copy_(finished)
        self.steps += 1
        return BeamStep(out.scores, tokens, out.parents)

    def done(self) -> bool:
        """Whether every beam is finished or has run out of tokens that may follow (waits for the GPU)."""
        return bool((self.finished | (self.scores == -math.inf)).all())

    def best(self, length_penalty: float = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
        """``(tokens [requests, steps], scores [requests])`` of every request's best hypothesis by score divided by
        its length to the power ``length_penalty``; the length counts up to and with ``eos_token``."""
        tokens = self.tokens[:, :self.steps].view(self.requests, self.beams, -1)
        length = torch.full_like(self.scores, float(max(1, self.steps)))
        if self.eos_token is not None and self.steps:
            ends = tokens == self.eos_token
            length = torch.where(ends.any(-1), ends.to(torch.int8).argmax(-1).float() + 1, length)
        ranked = self.scores / length**length_penalty
        at = ranked.argmax(1)
        rows = torch.arange(self.requests, device=at.device)
        return tokens[rows, at].clone(), ranked[rows, at]
