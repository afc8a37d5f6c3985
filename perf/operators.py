"""The measured calls of the beam-search decode path: products with a 4-bit head, the beam step, the state reorder.

One decode step of a beam search is: logits of every beam's hidden state under the LM head (here held in 4 bits with
group scales), the best continuations over beams and vocabulary, and the reordering of every per-beam state by the
parents of the chosen continuations.  ``run`` with ``own`` false computes each of the three in plain torch
operations; with ``own`` true it calls the framework.

4-bit layout (``qweight`` uint8 ``[tiles, chunks, 512]``).  A tile is 16 weight rows, a chunk 64 columns.  The 512
bytes of a (tile, chunk) are indexed ``[g 8][t 4][j 4][b1 2][b0 2]``; a byte holds rows ``16 tile + g`` (low nibble)
and ``16 tile + 8 + g`` (high nibble) of column ``64 chunk + 16 j + 8 b0 + 2 t + b1``.  ``scales`` (and ``zeros``,
uint8) are ``[tiles, groups, 8, 2]``: row ``g`` and row ``8 + g`` next to each other.  A weight is
``(q - zero) * scale`` with ``zero = 8`` where there are no zeros.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a small projection for one token: nothing but latency
        dict(name="int4_small_b1", op="int4", rows=2048, cols=1024, batch=1, group=128, zeros=False, x="bf16", out="bf16"),
        # the head of an 8B model, one sequence decoding alone, logits in fp32 as a sampler reads them
        dict(name="int4_head_b1", op="int4", rows=151936, cols=4096, batch=1, group=128, zeros=False, x="bf16", out="fp32"),
        # a vocabulary shard with a ragged last tile, five beams, asymmetric weights
        dict(name="int4_shard_b5", op="int4", rows=32776, cols=5376, batch=5, group=64, zeros=True, x="fp16", out="fp16"),
        # the head of a 70B model, four requests of four beams
        dict(name="int4_head_b16", op="int4", rows=128256, cols=8192, batch=16, group=128, zeros=True, x="bf16", out="bf16"),
        # one request of four beams, twice as many candidates as beams (the usual over-draw for finished sequences)
        dict(name="beam_one", op="beam", requests=1, beams=4, vocab=32000, candidates=8, dtype="fp32", masked="none", finished=False),
        # a ragged vocabulary in fp16 with a constraint mask of -inf that leaves some beams without a token
        dict(name="beam_odd", op="beam", requests=7, beams=5, vocab=32003, candidates=5, dtype="fp16", masked="inf", finished=False),
        # sixteen requests of four beams over a large vocabulary
        dict(name="beam_16x4", op="beam", requests=16, beams=4, vocab=151936, candidates=8, dtype="bf16", masked="none", finished=False),
        # a full batch: eight beams each, some finished, forbidden tokens at the type's lowest value
        dict(name="beam_64x8", op="beam", requests=64, beams=8, vocab=128256, candidates=16, dtype="bf16", masked="lowest", finished=True),
        # token histories of a small batch: a few kilobytes
        dict(name="reorder_tokens", op="reorder", requests=4, beams=4, outer=1, heads=1, steps=512, width=1, dtype="int64", layout="bhtd", lengths=False),
        # odd widths and step-major caches with ragged live lengths
        dict(name="reorder_odd", op="reorder", requests=6, beams=5, outer=5, heads=3, steps=777, width=41, dtype="bf16", layout="bthd", lengths=True),
        # keys and values of 32 layers, eight requests of four beams, 1k of 2k positions live on average
        dict(name="reorder_cache", op="reorder", requests=8, beams=4, outer=64, heads=8, steps=2048, width=64, dtype="bf16", layout="bhtd", lengths=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["int4", "int4", "beam", "beam", "reorder"])
    if kind == "int4":
        group = rng.choice([32, 64, 128])
        cols = max(1, _log_int(rng, 256, 16384) // group) * group
        rows = min(_log_int(rng, 64, 262208), 128256 * 7168 // cols)
        return dict(op="int4", rows=rows, cols=cols, batch=_log_int(rng, 1, 16), group=group, zeros=rng.random() < 0.5,
                    x=rng.choice(["bf16", "fp16"]), out=rng.choice(["bf16", "fp16", "fp32"]))
    if kind == "beam":
        beams = rng.randint(1, 12)
        vocab = _log_int(rng, 1000, 262208)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        requests = min(_log_int(rng, 1, 64), 56 * 8 * 128256 // (beams * vocab * (2 if dtype == "fp32" else 1)))
        return dict(op="beam", requests=requests, beams=beams, vocab=vocab, candidates=rng.choice([beams, 2 * beams]),
                    dtype=dtype, masked=rng.choice(["none", "inf", "lowest"]),
                    finished=rng.random() < 0.5)
    beams = rng.randint(2, 10)
    requests, outer, heads = _log_int(rng, 1, 16), _log_int(rng, 1, 64), rng.randint(1, 8)
    width = rng.choice([1, 41, 64, 80, 128])
    steps = max(1, min(_log_int(rng, 16, 8192), 8 * 4 * 64 * 8 * 2048 * 64 * 2 // (19 * requests * beams * outer * heads * width)))
    return dict(op="reorder", requests=requests, beams=beams, outer=outer, heads=heads, steps=steps, width=width,
                dtype=rng.choice(["bf16", "fp32", "int64"]), layout=rng.choice(["bhtd", "bthd"]), lengths=rng.random() < 0.7)


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    c = case
    if c["op"] == "int4":
        tiles, chunks, groups = -(-c["rows"] // 16), -(-c["cols"] // 64), c["cols"] // c["group"]
        dt = DTYPES[c["x"]]

        # nibbles of bell-shaped weights, two at a time
        nibble = lambda: (randn(tiles, chunks, 512) * 2.6 + 8).round_().clamp_(0, 15).to(torch.uint8)  # noqa: E731
        q = nibble() | (nibble() << 4)
        scales = ((0.5 + rand(tiles, groups, 8, 2)) * 0.008).to(dt)
        zeros = torch.randint(5, 12, (tiles, groups, 8, 2), generator=g, device="cuda", dtype=torch.uint8) if c["zeros"] else None
        x = randn(c["batch"], c["cols"]) * (1 + 15 * (rand(c["cols"]) < 0.002))  # a few large channels, as hidden states have
        return dict(case=c, x=x.to(dt), qweight=q, scales=scales, zeros=zeros)
    if c["op"] == "beam":
        R, K, V = c["requests"], c["beams"], c["vocab"]
        x = randn(R, K, V) * 2.2
        x += (rand(R, K, V) < 24 / V) * (6 + 5 * rand(R, K, V))  # the plausible continuations
        x = x.to(DTYPES[c["dtype"]])
        if c["masked"] != "none":
            low = -math.inf if c["masked"] == "inf" else torch.finfo(x.dtype).min
            x.masked_fill_(rand(R, K, V) < 0.4, low)
            dead = rand(R, K) < 0.1
            dead[:, 0] = False
            x.masked_fill_(dead[..., None], -math.inf)  # no allowed token left
        scores = -(8 * rand(R, K)).cumsum(1)
        done = (torch.arange(R * K, device="cuda").reshape(R, K) % 8 == 7) if c["finished"] else None
        return dict(case=c, logits=x, scores=scores, finished=done)
    R, K = c["requests"], c["beams"]
    shape = (c["outer"], R * K) + ((c["heads"], c["steps"]) if c["layout"] == "bhtd" else (c["steps"], c["heads"])) + (c["width"],)
    if c["dtype"] == "int64":
        state = torch.randint(0, 151936, shape, generator=g, device="cuda")
    else:
        state = torch.empty(shape, dtype=DTYPES[c["dtype"]], device="cuda").normal_(generator=g)
    parents = torch.randint(0, K, (R, K), generator=g, device="cuda")
    lengths = (rand(R) * c["steps"]).ceil().to(torch.int32) if c["lengths"] else None
    return dict(case=c, state=state, parents=parents, lengths=lengths)


# ---------------------------------------------------------------------------------------------- plain forms
def _rows_of_tiles(t, rows):
    """[tiles, groups, 8, 2] -> [rows, groups]."""
    return t.permute(0, 3, 2, 1).reshape(-1, t.shape[1])[:rows]


def _int4_plain(s):
    c = s["case"]
    tiles, chunks, _ = s["qweight"].shape
    q = s["qweight"].view(tiles, chunks, 8, 4, 4, 2, 2)  # g t j b1 b0
    q = torch.stack((q & 15, q >> 4), dim=1)  # tile h chunk g t j b1 b0
    q = q.permute(0, 1, 3, 2, 5, 7, 4, 6).reshape(tiles * 16, chunks * 64)[:c["rows"], :c["cols"]]
    w = q.float().view(c["rows"], -1, c["group"])
    w = w - (8.0 if s["zeros"] is None else _rows_of_tiles(s["zeros"], c["rows"]).float()[..., None])
    w = w * _rows_of_tiles(s["scales"], c["rows"]).float()[..., None]
    return (s["x"].float() @ w.view(c["rows"], c["cols"]).T).to(DTYPES[c["out"]])


def _beam_plain(s):
    c = s["case"]
    R, K, V, N = c["requests"], c["beams"], c["vocab"], c["candidates"]
    # which of two close candidates comes first is a matter of the last bits: everything here in 64
    x = s["logits"].double().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    top = x.amax(-1, keepdim=True)
    score = s["scores"].double()[..., None]
    usable = top.isfinite() & score.isfinite()
    shifted = x - torch.where(usable, top, torch.zeros_like(top))
    total = score + (shifted - shifted.exp().sum(-1, keepdim=True).log())
    total = torch.where(usable, total, torch.full_like(total, -math.inf))
    if s["finished"] is not None:  # a finished beam goes on as it is: one candidate, the padding token 0
        alone = torch.full_like(total, -math.inf)
        alone[..., 0] = score[..., 0]
        total = torch.where(s["finished"][..., None], alone, total)
    total = total.view(R, K * V)
    # the N largest, of equal ones those of the lowest index
    last = total.topk(N, dim=1).values[:, -1:]
    above, equal = total > last, total == last
    taken = above | (equal & (equal.cumsum(1) <= N - above.sum(1, keepdim=True)))
    at = torch.where(taken, torch.arange(K * V, device=total.device), K * V).topk(N, dim=1, largest=False, sorted=True).values
    value, order = total.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    none = value == -math.inf
    slot = torch.arange(N, device=total.device).clamp_max(K - 1).expand(R, N)
    return (value.float(), torch.where(none, torch.full_like(at, -1), at % V), torch.where(none, slot, at // V))


def _reorder_plain(s):
    c, state = s["case"], s["state"]
    R, K = c["requests"], c["beams"]
    rows = (torch.arange(R, device="cuda")[:, None] * K + s["parents"]).flatten()
    moved = state.index_select(1, rows)
    if s["lengths"] is not None:
        live = torch.arange(c["steps"], device="cuda") < s["lengths"].repeat_interleave(K)[:, None]  # [R * K, steps]
        live = live[:, None, :, None] if c["layout"] == "bhtd" else live[:, :, None, None]
        moved = torch.where(live, moved, state)
    return state.copy_(moved)


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    c = state["case"]
    if own:
        import flashsampling_b200 as fs

        if c["op"] == "int4":
            w = fs.Int4Weight(state["qweight"], state["scales"], state["zeros"], rows=c["rows"], cols=c["cols"])
            return fs.int4_linear(state["x"], w, out_dtype=DTYPES[c["out"]])
        if c["op"] == "beam":
            step = fs.beam_search_step(state["logits"], state["scores"], num_candidates=c["candidates"],
                                       finished=state["finished"], pad_token=0)
            return step.scores, step.tokens, step.parents
        fs.reorder_beams(state["state"], state["parents"], dim=1, lengths=state["lengths"],
                         length_dim=3 if c["layout"] == "bhtd" else 2)
        return state["state"]
    return {"int4": _int4_plain, "beam": _beam_plain, "reorder": _reorder_plain}[c["op"]](state)


def work(case):
    c = case
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "int64": 8}
    if c["op"] == "int4":
        params = c["rows"] * c["cols"]
        per_group = 2 + (1 if c["zeros"] else 0)
        return {"bytes": params / 2 + params // c["group"] * per_group + c["batch"] * (c["cols"] * 2 + c["rows"] * size[c["out"]]),
                "flops": 2 * params * c["batch"]}
    if c["op"] == "beam":
        beams = c["requests"] * c["beams"]
        live = beams - beams // 8 if c["finished"] else beams
        return {"bytes": live * c["vocab"] * size[c["dtype"]] + beams * 5 + c["requests"] * c["candidates"] * 20,
                "flops": 4 * live * c["vocab"]}
    K = c["beams"]
    written = K - 1  # of K beams whose parent is any of the K alike, one keeps its own state
    read = K * (1 - (1 - 1 / K) ** (K - 1))  # beams that another one takes over
    row = c["outer"] * c["heads"] * c["steps"] * c["width"] * size[c["dtype"]] * (0.5 if c["lengths"] else 1)
    return {"bytes": c["requests"] * ((read + written) * row + 8 * K), "flops": 0}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "reorder":  # values are moved, none is computed: beam by beam
        out, K = s["state"].clone(), c["beams"]
        for r in range(c["requests"]):
            n = c["steps"] if s["lengths"] is None else int(s["lengths"][r])
            for k in range(K):
                src = s["state"][:, r * K + int(s["parents"][r, k])]
                if c["layout"] == "bhtd":
                    out[:, r * K + k, :, :n] = src[:, :, :n]
                else:
                    out[:, r * K + k, :n] = src[:, :n]
        return out
    if c["op"] == "int4":
        # nibble by nibble from the layout's definition: the byte of (row, column) and its half
        rows, cols = torch.arange(c["rows"], device="cuda"), torch.arange(c["cols"], device="cuda")
        k = cols % 16
        byte = (k % 8 // 2) * 16 + (cols % 64 // 16) * 4 + (k % 2) * 2 + k // 8
        x = s["x"].double()
        out = torch.empty(c["batch"], c["rows"], dtype=torch.float64, device="cuda")
        flat = s["qweight"].view(-1)
        for r0 in range(0, c["rows"], 8192):
            r = rows[r0:r0 + 8192, None]
            at = (r // 16 * s["qweight"].shape[1] + cols // 64) * 512 + r % 8 * 64 + byte
            q = (flat[at] >> (r % 16 // 8 * 4)) & 15
            grp = cols // c["group"]
            scale = s["scales"][r // 16, grp, r % 8, r % 16 // 8].double()
            zero = 8.0 if s["zeros"] is None else s["zeros"][r // 16, grp, r % 8, r % 16 // 8].double()
            out[:, r0:r0 + 8192] = x @ ((q.double() - zero) * scale).T
        return out
    R, K, V, N = c["requests"], c["beams"], c["vocab"], c["candidates"]
    scores = torch.full((R, N), -math.inf, dtype=torch.float64, device="cuda")
    tokens = torch.full((R, N), -1, dtype=torch.int64, device="cuda")
    parents = torch.arange(N, device="cuda").clamp_max(K - 1).repeat(R, 1)
    for r in range(R):
        found = []  # (value, parent, token), beam by beam
        for k in range(K):
            base = float(s["scores"][r, k])
            if s["finished"] is not None and bool(s["finished"][r, k]):
                found.append((torch.tensor([base], dtype=torch.float64, device="cuda"), k, torch.zeros(1, dtype=torch.int64, device="cuda")))
                continue
            lp = s["logits"][r, k].double()
            if not bool(lp.isfinite().any()):
                continue
            lp = lp.log_softmax(0)
            value, token = lp.sort(descending=True, stable=True)
            n = min(N, int((value > -math.inf).sum()))
            found.append((base + value[:n], k, token[:n]))
        if not found:
            continue
        value = torch.cat([f[0] for f in found])
        parent = torch.cat([torch.full_like(f[2], f[1]) for f in found])
        token = torch.cat([f[2] for f in found])
        value, order = value.sort(descending=True, stable=True)
        n = min(N, value.numel())
        scores[r, :n], tokens[r, :n], parents[r, :n] = value[:n], token[order][:n], parent[order][:n]
    return scores, tokens, parents
