"""Operators for the rows and scores of a language model, as timed cases: rows held in four bits with group scales (encoding, and
products with a few vectors), the selection of a beam search, and the reordering of its states.

``listed()`` holds the fixed cases, ``draw(rng)`` one more case of the same ranges, ``prepare(case, seed)`` makes the inputs a program
holds before the call, ``run(state)`` is one call, ``work(case)`` the bytes and operations it cannot do without and ``exact(case, seed)``
the same results in 64 bits.  With ``own`` false ``run`` computes the operators with elementary torch operations, with ``own`` true it
calls this package.  All data are synthetic.
"""
import math

import numpy as np
import torch

own = False

_DEVICE = []


def _device():
    """One device object for the process, as a program holds it."""
    import vectorstorekit_b200 as vsk
    if not _DEVICE:
        _DEVICE.append(vsk.CUDAAcceleratorStrategy(0).initialize())
    return _DEVICE[0]


_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases ---------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token through one square projection: the smallest call of a decoding step
        dict(name="product_one_token", family="product", rows=4_096, dim=4_096, queries=1, group=64, symmetric=True, x="f16", y="f16"),
        # one fp32 query against a large store of text embeddings, bound by the bytes of the rows
        dict(name="product_one_query", family="product", rows=1_000_000, dim=768, queries=1, group=32, symmetric=False, x="f32", y="f32"),
        # the output head under the beams of a search: many rows, tens of vectors
        dict(name="product_head_beams", family="product", rows=131_072, dim=2_048, queries=32, group=128, symmetric=True, x="bf16",
             y="f32"),
        # a small batch over rows whose length no tile divides
        dict(name="product_odd_batch", family="product", rows=50_001, dim=1_000, queries=5, group=64, symmetric=False, x="f16", y="f32"),
        # a block of new embeddings on its way into four bits, and back
        dict(name="encode_small", family="encode", rows=10_000, dim=384, group=64, symmetric=True, x="f16"),
        dict(name="encode_large", family="encode", rows=100_000, dim=768, group=32, symmetric=False, x="f32"),
        # one prompt, four beams: the smallest selection
        dict(name="select_one", family="select", batch=1, beams=4, vocab=32_768, k=8, dtype="f32", normalize=True, masked=0.0,
             finished=0.0, pad=0),
        # several prompts with finished beams and forbidden tokens, rows inside wider ones, an odd vocabulary
        dict(name="select_odd", family="select", batch=7, beams=5, vocab=50_001, k=10, dtype="f16", normalize=True, masked=0.3,
             finished=0.2, pad=15),
        # chains of retrievals: every chain brings the hundred rows a search has found for it, with their scores
        dict(name="select_chains", family="select", batch=1_000, beams=8, vocab=100, k=8, dtype="f32", normalize=False, masked=0.1,
             finished=0.05, pad=0),
        # a large batch over a large vocabulary
        dict(name="select_large", family="select", batch=32, beams=8, vocab=131_072, k=16, dtype="bf16", normalize=True, masked=0.0,
             finished=0.0, pad=0),
        # a short cache whose lost beams take copies of the ones that live on, in place
        dict(name="reorder_small", family="reorder", batch=2, beams=4, tensors=4, heads=8, steps=256, width=64, dtype="f16",
             in_place=True),
        # the caches of a large batch into their second set of buffers, prompts of different lengths
        dict(name="reorder_large", family="reorder", batch=8, beams=8, tensors=8, heads=8, steps=1_024, width=128, dtype="bf16",
             in_place=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["product", "product", "product", "encode", "select", "select", "select", "reorder"])
    if family == "product":
        queries = rng.choice([1, _log(rng, 1, 64)])
        dim = _log(rng, 64, 8_192)
        rows = _log(rng, 1_000, 1_000_000)
        # neither more bytes nor more products than the largest listed ones
        rows = max(64, min(rows, int(7.6e8 / dim), int(8.5e9 / (dim * queries))))
        x = rng.choice(["f32", "f16", "bf16"])
        return dict(family="product", rows=rows, dim=dim, queries=queries, group=rng.choice([32, 64, 128]),
                    symmetric=rng.random() < 0.5, x=x, y=rng.choice(["f32", x]))
    if family == "encode":
        dim = _log(rng, 32, 4_096)
        rows = max(100, min(_log(rng, 1_000, 500_000), int(7.6e7 / dim)))
        return dict(family="encode", rows=rows, dim=dim, group=rng.choice([32, 64, 128]), symmetric=rng.random() < 0.5,
                    x=rng.choice(["f32", "f16", "bf16"]))
    if family == "select":
        beams = rng.choice([1, _log(rng, 1, 32)])
        vocab = rng.choice([_log(rng, 20, 2_000), _log(rng, 2_000, 262_144), _log(rng, 2_000, 262_144)])
        batch = max(1, min(_log(rng, 1, 1_000), int(3.3e7 / (beams * vocab))))
        return dict(family="select", batch=batch, beams=beams, vocab=vocab, k=_log(rng, 1, 64), dtype=rng.choice(["f32", "f16", "bf16"]),
                    normalize=rng.random() < 0.7, masked=rng.choice([0.0, 0.3, 0.95]), finished=rng.choice([0.0, 0.2]),
                    pad=rng.choice([0, 0, 7]))
    beams = _log(rng, 2, 32)
    heads, steps, width = _log(rng, 1, 16), _log(rng, 16, 2_048), rng.choice([64, 80, 128, 33])
    batch = max(1, min(_log(rng, 1, 16), int(6.7e7 / (beams * heads * steps * width))))
    tensors = max(1, min(_log(rng, 1, 32), int(5.3e8 / (batch * beams * heads * steps * width))))
    return dict(family="reorder", batch=batch, beams=beams, tensors=tensors, heads=heads, steps=steps, width=width,
                dtype=rng.choice(["f32", "f16", "bf16"]) if tensors * batch * beams * heads * steps * width < 2.6e8 else "bf16",
                in_place=rng.random() < 0.5)


# ---- rows in four bits: the plain form of the codec ------------------------------------------------------------------

def _columns(dim, group, device):
    """Column numbers of the groups; a short last group repeats its last column, which changes no minimum or maximum."""
    groups = -(-dim // group)
    return torch.arange(groups * group, device=device).clamp(max=dim - 1).view(groups, group)


def _encode(rows, group, symmetric):
    """-> (codes as whole numbers -8 .. 7 [n][dim], scales [n][groups], middles [n][groups] or None)"""
    dim = rows.shape[1]
    cols = _columns(dim, group, rows.device)
    x = rows.double()
    g = x[:, cols]
    if symmetric:
        step = (g.abs().amax(2) / 7.0).float().clamp(max=65504.0).half()
        mid = None
        away = x
    else:
        lo, hi = g.amin(2), g.amax(2)
        step = ((hi - lo) / 15.0).float().clamp(max=65504.0).half()
        mid = (lo + 8.0 * step.double()).float().clamp(-65504.0, 65504.0).half()
        away = x - mid.double().repeat_interleave(group, 1)[:, :dim]
    wide = step.double().repeat_interleave(group, 1)[:, :dim]
    codes = torch.where(wide > 0, away / wide, 0.0).round().clamp(-8, 7)
    return codes.to(torch.int8), step, mid


def _pack(codes):
    """Two codes a byte, the even column in the low half."""
    n, dim = codes.shape
    u = (codes + 8).to(torch.uint8)
    if dim % 2:
        u = torch.cat([u, torch.full((n, 1), 8, dtype=torch.uint8, device=u.device)], 1)
    return u[:, 0::2] | (u[:, 1::2] << 4)


def _values(codes, step, mid, dim, group):
    """The values that packed codes stand for, in fp32."""
    u = torch.stack([codes & 15, codes >> 4], 2).flatten(1)[:, :dim]
    out = (u.float() - 8.0) * step.float().repeat_interleave(group, 1)[:, :dim]
    return out if mid is None else out + mid.float().repeat_interleave(group, 1)[:, :dim]


# ---- inputs ------------------------------------------------------------------------------------------------------

_PIECE = 1 << 24   # values encoded at a time


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, shape, dtype):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=gen).to(dtype)


def _rows(gen, n, dim):
    """Rows of embeddings or weights: columns of different spreads around a small mean of their own."""
    spread = torch.empty(dim, device="cuda").uniform_(0.3, 1.7, generator=gen) / math.sqrt(dim)
    shift = torch.empty(dim, device="cuda").normal_(generator=gen) * (0.2 / math.sqrt(dim))
    return torch.empty((n, dim), device="cuda").normal_(generator=gen) * spread + shift


def prepare(case, seed):
    gen = _generator(seed)
    family = case["family"]
    s = {"case": case}
    if family == "product":
        n, dim, group = case["rows"], case["dim"], case["group"]
        # rows of a whole number of 16-byte pieces, as the encoder lays them out
        codes = torch.zeros((n, -(-dim // 32) * 16), dtype=torch.uint8, device="cuda")[:, : -(-dim // 2)]
        scales = torch.empty((n, -(-dim // group)), dtype=torch.float16, device="cuda")
        middles = None if case["symmetric"] else torch.empty_like(scales)
        piece = max(1, _PIECE // dim)
        for b in range(0, n, piece):
            c, step, mid = _encode(_rows(gen, min(piece, n - b), dim), group, case["symmetric"])
            codes[b:b + piece] = _pack(c)
            scales[b:b + piece] = step
            if mid is not None:
                middles[b:b + piece] = mid
        s.update(codes=codes, scales=scales, middles=middles, x=_normal(gen, (case["queries"], dim), _TYPES[case["x"]]))
    elif family == "encode":
        s.update(rows=_rows(gen, case["rows"], case["dim"]).to(_TYPES[case["x"]]))
    elif family == "select":
        b, w, v = case["batch"], case["beams"], case["vocab"]
        wide = _normal(gen, (b, w, v + case["pad"]), torch.float32)
        if case["normalize"]:
            wide *= 3.0
        if case["masked"]:
            wide[torch.rand(wide.shape, device="cuda", generator=gen) < case["masked"]] = float("-inf")
        scores = -torch.rand((b, w), device="cuda", generator=gen).mul_(20.0).sort(dim=1)[0]
        finished = torch.rand((b, w), device="cuda", generator=gen) < case["finished"] if case["finished"] else None
        s.update(logits=wide.to(_TYPES[case["dtype"]])[:, :, :v], scores=scores, finished=finished, k=case["k"], end=v // 2)
    else:
        b, w = case["batch"], case["beams"]
        shape = (b * w, case["heads"], case["steps"], case["width"])
        states = [_normal(gen, shape, _TYPES[case["dtype"]]) for _ in range(case["tensors"])]
        parents = torch.randint(0, w, (b, w), device="cuda", generator=gen)
        if case["in_place"]:
            # beams that somebody continues stay where they are, the others' places take copies
            alive = torch.zeros((b, w), dtype=torch.bool, device="cuda").scatter_(1, parents, True)
            parents = torch.where(alive, torch.arange(w, device="cuda"), parents)
        lengths = torch.randint(1, case["steps"] + 1, (b,), device="cuda", generator=gen)
        lengths[0] = case["steps"]
        s.update(states=states, parents=parents, lengths=lengths)
        s.update(out=states if case["in_place"] else [torch.zeros_like(t) for t in states])
    return s


# ---- one call ----------------------------------------------------------------------------------------------------

def _select(logits, scores, finished, end, k, normalize):
    b, w, v = logits.shape
    none = float("-inf")
    x = logits.double()
    x = torch.where(x.isnan(), none, x)
    live = scores.isfinite()
    if normalize:
        top = x.amax(2, keepdim=True)
        total = (x - torch.where(top.isfinite(), top, 0.0)).exp().sum(2, keepdim=True).log() + top
        ok = (top.isfinite() & ~logits.isnan().any(2, keepdim=True)) & live[:, :, None]
        x = torch.where(ok, x - total, none)
    else:
        x = torch.where(live[:, :, None], x, none)
    x = x + scores.double().where(live, torch.zeros((), dtype=torch.float64, device=x.device))[:, :, None]
    if finished is not None:
        x = torch.where(finished[:, :, None], none, x)
        x[:, :, end] = torch.where(finished & live, scores.double(), x[:, :, end])
    x = x.view(b, w * v)
    if w * v < k:
        x = torch.cat([x, torch.full((b, k - w * v), none, dtype=x.dtype, device=x.device)], 1)
    last = x.topk(k, dim=1)[0][:, -1:]
    above, level = x > last, x == last
    taken = above | (level & (level.cumsum(1) <= k - above.sum(1, keepdim=True)))
    at = taken.nonzero()[:, 1].view(b, k)                                  # ascending
    best, order = x.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    found = best > none
    return best.float(), torch.where(found, at // v, -1), torch.where(found, at % v, -1)


def _reorder(states, parents, lengths, out):
    b, w = parents.shape
    rows = (torch.arange(b, device=parents.device)[:, None] * w + parents).view(-1)
    steps = states[0].shape[2]
    live = (torch.arange(steps, device=parents.device) < lengths[:, None]).repeat_interleave(w, 0)[:, None, :, None]
    return [o.copy_(torch.where(live, t[rows], o)) for t, o in zip(states, out)]


def run(state):
    case = state["case"]
    family = case["family"]
    if own:
        import vectorstorekit_b200 as vsk
        dev = _device()
        if family == "product":
            quantizer = vsk.Int4Quantizer(dev, groupSize=case["group"], symmetric=case["symmetric"])
            return quantizer.product(state["x"], state["codes"], state["scales"], state["middles"], out_dtype=_TYPES[case["y"]])
        if family == "encode":
            quantizer = vsk.Int4Quantizer(dev, groupSize=case["group"], symmetric=case["symmetric"])
            codes, scales, middles = quantizer.quantizeBatch(state["rows"])
            values = quantizer.dequantizeBatch(codes, scales, middles, case["dim"])
            return (values, scales) if middles is None else (values, scales, middles)
        engine = vsk.CUDAAccelerationEngine(dev)
        if family == "select":
            return engine.selectBeams(state["logits"], state["scores"], state["k"], normalize=case["normalize"],
                                      finished=state["finished"], end_token=state["end"])
        return engine.reorderStates(state["states"], state["parents"], lengths=state["lengths"], time_axis=2,
                                    out=None if case["in_place"] else state["out"])
    if family == "product":
        w = _values(state["codes"], state["scales"], state["middles"], case["dim"], case["group"])
        return (state["x"].float() @ w.T).to(_TYPES[case["y"]])
    if family == "encode":
        codes, scales, middles = _encode(state["rows"], case["group"], case["symmetric"])
        values = _values(_pack(codes), scales, middles, case["dim"], case["group"])
        return (values, scales) if middles is None else (values, scales, middles)
    if family == "select":
        return _select(state["logits"], state["scores"], state["finished"], state["end"], state["k"], case["normalize"])
    return _reorder(state["states"], state["parents"], state["lengths"], state["out"])


# ---- what a pass cannot do without -------------------------------------------------------------------------------

_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    family = case["family"]
    if family in ("product", "encode"):
        n, dim = case["rows"], case["dim"]
        held = n * (-(-dim // 2)) + n * (-(-dim // case["group"])) * (2.0 if case["symmetric"] else 4.0)
        if family == "product":
            io = case["queries"] * (dim * _BYTES[case["x"]] + n * _BYTES[case["y"]])
            return {"bytes": held + io, "flops": 2.0 * n * dim * case["queries"]}
        # rows in, codes and scales out; codes and scales in, values out
        return {"bytes": n * dim * (_BYTES[case["x"]] + 4.0) + 2.0 * held, "flops": 8.0 * n * dim}
    if family == "select":
        rows = case["batch"] * case["beams"] * (1.0 - case["finished"])
        return {"bytes": rows * case["vocab"] * _BYTES[case["dtype"]] + 20.0 * case["batch"] * case["k"],
                "flops": rows * case["vocab"] * (4.0 if case["normalize"] else 1.0)}
    w = case["beams"]
    row = case["tensors"] * case["heads"] * case["width"] * _BYTES[case["dtype"]] * (case["steps"] + 1) / 2.0
    # of w random parents w (1 - (1 - 1/w)^w) are distinct: those rows are read, and all are written, or in place the others
    distinct = w * (1.0 - (1.0 - 1.0 / w) ** w)
    if case["in_place"]:
        moved = w - distinct
        return {"bytes": case["batch"] * row * (min(moved, distinct) + moved), "flops": 0.0}
    return {"bytes": case["batch"] * row * (distinct + w), "flops": 0.0}


# ---- the same in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    family = case["family"]
    if family == "product":
        n, dim, group = case["rows"], case["dim"], case["group"]
        x, half = s["x"].double(), torch.arange(-8, 8, dtype=torch.float64, device="cuda")
        of = torch.arange(dim, device="cuda") // group
        y = torch.empty((case["queries"], n), dtype=torch.float64, device="cuda")
        piece = max(1, _PIECE // dim)
        for b in range(0, n, piece):
            packed = s["codes"][b:b + piece].long()
            w = torch.empty((packed.shape[0], 2 * packed.shape[1]), dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = half[packed % 16], half[packed // 16]
            w = w[:, :dim] * s["scales"][b:b + piece].double()[:, of]
            if s["middles"] is not None:
                w += s["middles"][b:b + piece].double()[:, of]
            y[:, b:b + piece] = torch.einsum("qd,nd->qn", x, w)
        return y.cpu().numpy()
    if family == "encode":
        rows, group = s["rows"].double().cpu().numpy(), case["group"]
        n, dim = rows.shape
        starts = np.arange(0, dim, group)
        width = np.diff(np.append(starts, dim))
        hi, lo = np.maximum.reduceat(rows, starts, axis=1), np.minimum.reduceat(rows, starts, axis=1)
        if case["symmetric"]:
            step, mid = np.maximum(hi, -lo) / 7.0, np.zeros_like(lo)
        else:
            step, mid = (hi - lo) / 15.0, None
        step = np.minimum(step.astype(np.float32), np.float32(65504)).astype(np.float16)
        if mid is None:
            mid = np.clip((lo + 8.0 * step.astype(np.float64)).astype(np.float32), -65504, 65504).astype(np.float16)
        wide, middle = (np.repeat(a.astype(np.float64), width, axis=1) for a in (step, mid))
        with np.errstate(divide="ignore", invalid="ignore"):
            codes = np.clip(np.rint(np.where(wide > 0, (rows - middle) / wide, 0.0)), -8, 7)
        values = codes * wide + middle
        held = (values, step.astype(np.float64))
        return held if case["symmetric"] else held + (mid.astype(np.float64),)
    if family == "select":
        logits, scores = s["logits"].float().cpu().numpy(), s["scores"].double().cpu().numpy()
        over = None if s["finished"] is None else s["finished"].cpu().numpy()
        b, w, v = logits.shape
        k = s["k"]
        best, beams, tokens = np.full((b, k), -np.inf), np.full((b, k), -1, np.int64), np.full((b, k), -1, np.int64)
        for i in range(b):
            l = logits[i].astype(np.float64)
            if case["normalize"]:
                top = l.max(1, keepdims=True)
                with np.errstate(invalid="ignore", divide="ignore"):
                    l = l - (top + np.log(np.exp(l - top).sum(1, keepdims=True)))
            l += scores[i][:, None]
            if over is not None:
                l[over[i]] = -np.inf
                l[over[i], s["end"]] = scores[i][over[i]]
            flat = np.where(np.isnan(l), -np.inf, l).reshape(-1)
            near = np.argpartition(-flat, k - 1)[:k] if k < flat.size else np.arange(flat.size)
            near = np.nonzero((flat >= flat[near].min()) & (flat > -np.inf))[0]
            near = near[np.argsort(-flat[near], kind="stable")][:k]
            best[i, :near.size], beams[i, :near.size], tokens[i, :near.size] = flat[near], near // v, near % v
        return best, beams, tokens
    return None                          # rows are moved, nothing is computed
