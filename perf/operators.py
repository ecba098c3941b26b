"""Performance cases of the decoding operators: products of a few rows with 4-bit weights, the best `keep` continuations
of every beam search (a max-plus step with back-pointers), and the reordering of the beams' states by those back-pointers.

`listed()` names twelve calls that stand for the whole range, `draw(rng)` makes further ones of the same ranges, `run`
computes a case in elementary torch operations or, where `own` is true, through this package, and `exact` computes it
from the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

TORCH_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def q4(m, n, k, group, x="bf16", y="bf16", scale="bf16", zeros=False):
    """Y = X W^T: X is m x k, W n x k in 4 bits with a scale (and a zero point) for every `group` values along k."""
    return {"kind": "q4", "m": m, "n": n, "k": k, "group": group, "x": x, "y": y, "scale": scale, "zeros": zeros}


def beam(batch, beams, vocab, keep, dtype="f32", normalise=True, finished=False, masked=False, first=False):
    """The best `keep` of beams x vocab continuations of each of `batch` searches.  normalise: the inputs are logits, not
    log-probabilities.  finished: some beams have ended.  masked: half of the vocabulary is ruled out (-inf).  first: the
    first step of a search, where one beam alone holds a prefix."""
    return {"kind": "beam", "batch": batch, "beams": beams, "vocab": vocab, "keep": keep, "dtype": dtype,
            "normalise": normalise, "finished": finished, "masked": masked, "first": first}


def reorder(batch, beams, heads, positions, dim, tensors, dtype="bf16", in_place=True, ragged=True):
    """`tensors` state tensors of batch x beams x heads x positions x dim follow the beams they belong to.  ragged: each
    search has its own number of positions in use."""
    return {"kind": "reorder", "batch": batch, "beams": beams, "heads": heads, "positions": positions, "dim": dim,
            "tensors": tensors, "dtype": dtype, "in_place": in_place, "ragged": ragged}


def listed():
    return [
        # The smallest product of a decoding step: a low-rank or key/value projection of one token.
        dict(q4(1, 1024, 1024, 64, "f16", "f16", "f16"), name="q4_1x1024x1024_f16"),
        # One token through a square layer of an ordinary size.
        dict(q4(1, 4096, 4096, 128), name="q4_1x4096x4096_bf16"),
        # The four beams of one search through a wide layer, weights with zero points.
        dict(q4(4, 14336, 4096, 128, zeros=True), name="q4_4x14336x4096_bf16_zeros"),
        # Single-precision activations, odd sizes, groups of 32 with a short last one.
        dict(q4(3, 5003, 2999, 32, "f32", "f32", "f16", zeros=True), name="q4_3x5003x2999_f32"),
        # Eight searches of four beams through a large layer.
        dict(q4(32, 8192, 8192, 128, "f16", "f16", "f16"), name="q4_32x8192x8192_f16"),
        # The projection onto the vocabulary, whose logits the next operator takes.
        dict(q4(8, 128000, 4096, 128, "bf16", "f32"), name="q4_8x128000x4096_logits"),
        # One search, log-probabilities at hand: latency counts.
        dict(beam(1, 4, 32000, 8, normalise=False), name="beam_1x4x32000_f32"),
        # Odd sizes, half precision, ended beams, tokens that a grammar rules out.
        dict(beam(5, 7, 50021, 14, "f16", finished=True, masked=True), name="beam_5x7x50021_f16_masked"),
        # A server's batch: 32 searches of four beams over a large vocabulary, logits in 16 bits.
        dict(beam(32, 4, 128000, 8, "bf16", finished=True), name="beam_32x4x128000_bf16"),
        # A wide search over many inputs, logits in 32 bits.
        dict(beam(64, 16, 64000, 32), name="beam_64x16x64000_f32"),
        # Recurrent states of one search, from one set of buffers into another: latency counts.
        dict(reorder(1, 4, 8, 1, 4096, 8, "f32", in_place=False, ragged=False), name="reorder_recurrent_f32"),
        # The cached keys and values of eight layers, in place.
        dict(reorder(4, 4, 8, 2048, 128, 16), name="reorder_cache_bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number from [lo, hi], spread evenly over its logarithm; odd ones as likely as even ones."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("q4", "q4", "q4", "beam", "beam", "reorder"))
    if kind == "q4":
        m, n, k = _log(rng, 1, 32), _log(rng, 64, 32768), _log(rng, 64, 16384)
        if rng.random() < 0.6:       # rows of the weights start on 16-byte boundaries
            k = max(64, k // 32 * 32)
        x = rng.choice(("bf16", "f16", "f32"))
        return q4(m, n, k, rng.choice((32, 64, 128)), x, rng.choice((x, "f32")), rng.choice((x, "f16", "bf16", "f32")),
                  rng.random() < 0.5)
    if kind == "beam":
        beams = _log(rng, 1, 16)
        batch = _log(rng, 1, 64)
        vocab = _log(rng, 1000, min(150000, 60_000_000 // (beams * batch)))
        return beam(batch, beams, vocab, min(32, rng.choice((beams, 2 * beams, 2 * beams + 1))),
                    rng.choice(("f32", "f16", "bf16")), rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.3,
                    rng.random() < 0.2)
    beams, batch, heads = _log(rng, 2, 16), _log(rng, 1, 8), _log(rng, 1, 16)
    dim, tensors = rng.choice((64, 80, 96, 128)), _log(rng, 1, 32)
    positions = _log(rng, 1, max(1, min(4096, 500_000_000 // (beams * batch * heads * dim * tensors))))
    return reorder(batch, beams, heads, positions, dim, tensors, rng.choice(("bf16", "f32")), rng.random() < 0.6,
                   rng.random() < 0.6)


# ---- inputs ---------------------------------------------------------------------------------------------------
def _prepare_q4(case, g):
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    groups = -(-k // group)
    # weights of a layer keep the size of its inputs: 4-bit steps of about 1 / (4 sqrt(k))
    scales = (0.5 + torch.rand(n, groups, generator=g, device="cuda")) / (4 * math.sqrt(k))
    zeros = None
    if case["zeros"]:
        zeros = torch.randint(4, 12, (n, groups), generator=g, device="cuda", dtype=torch.uint8)
    return {"X": torch.randn(m, k, generator=g, device="cuda").to(TORCH_DTYPE[case["x"]]),
            "W": torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.uint8),
            "scales": scales.to(TORCH_DTYPE[case["scale"]]), "zeros": zeros,
            "Y": torch.empty(m, n, device="cuda", dtype=TORCH_DTYPE[case["y"]])}


def _prepare_beam(case, g):
    batch, beams, vocab, keep = case["batch"], case["beams"], case["vocab"], case["keep"]
    logits = torch.randn(batch, beams, vocab, generator=g, device="cuda").mul_(2.5)
    if case["masked"]:
        logits.masked_fill_(torch.rand(vocab, generator=g, device="cuda") < 0.5, -math.inf)
    if not case["normalise"]:
        logits = torch.log_softmax(logits, dim=-1)
    scores = -4 * torch.rand(batch, beams, generator=g, device="cuda") - 10
    if case["first"]:
        scores[:, 1:] = -math.inf
    finished = None
    if case["finished"]:
        finished = (torch.rand(batch, beams, generator=g, device="cuda") < 0.15).to(torch.uint8)
    return {"logits": logits.to(TORCH_DTYPE[case["dtype"]]), "scores": scores, "finished": finished, "end_token": 2,
            "out_scores": torch.empty(batch, keep, device="cuda"),
            "parents": torch.empty(batch, keep, device="cuda", dtype=torch.int32),
            "tokens": torch.empty(batch, keep, device="cuda", dtype=torch.int32)}


def _survivors(beams):
    """How many beams of a search have a continuation among the kept ones; the others are dropped."""
    return max(1, (5 * beams + 7) // 8)


def _lengths(case):
    """Positions in use of each search of a padded batch."""
    batch, positions = case["batch"], case["positions"]
    return [positions - positions * b // (2 * batch) if case["ragged"] else positions for b in range(batch)]


def _prepare_reorder(case, g):
    batch, beams = case["batch"], case["beams"]
    shape = (batch, beams, case["heads"], case["positions"], case["dim"])
    dtype = TORCH_DTYPE[case["dtype"]]
    src = [torch.randn(shape, generator=g, device="cuda", dtype=dtype) for _ in range(case["tensors"])]
    # the beams that live on, then repetitions of them, in an order of their own for each search
    live = torch.rand(batch, beams, generator=g, device="cuda").argsort(dim=1)
    live = live[:, torch.arange(beams, device="cuda") % _survivors(beams)]
    order = torch.rand(batch, beams, generator=g, device="cuda").argsort(dim=1)
    return {"src": src, "dst": src if case["in_place"] else [torch.zeros_like(t) for t in src],
            "parents": live.gather(1, order).to(torch.int32),
            "lengths": torch.tensor(_lengths(case), device="cuda", dtype=torch.int32) if case["ragged"] else None}


PREPARE = {"q4": _prepare_q4, "beam": _prepare_beam, "reorder": _prepare_reorder}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(PREPARE[case["kind"]](case, g), case=case)
    if own:
        # the operator object a decoding loop sets up once for its buffers, as with Srgemm.initialize() and run()
        state["op"] = _operator(case, state)
    return state


# ---- this package's operators -----------------------------------------------------------------------------------
def _operator(case, s):
    from cuasr_b200 import (BeamArguments, BeamStep, DType, Q4Arguments, Q4Product, ReorderArguments, ReorderStates, Status,
                            state_view)
    dtype = {"f32": DType.F32, "f16": DType.F16, "bf16": DType.BF16}
    workspace = None
    if case["kind"] == "q4":
        m, n, k = case["m"], case["n"], case["k"]
        zeros = (None, 0) if s["zeros"] is None else (s["zeros"], s["zeros"].shape[1])
        op = Q4Product(dtype[case["x"]], dtype[case["y"]], dtype[case["scale"]], case["group"])
        args = Q4Arguments((m, n, k), (s["X"], k), (s["W"], s["W"].shape[1]), (s["scales"], s["scales"].shape[1]), (s["Y"], n),
                           zeros)
    elif case["kind"] == "beam":
        beams, vocab, keep = case["beams"], case["vocab"], case["keep"]
        op = BeamStep(dtype[case["dtype"]], normalise=case["normalise"])
        args = BeamArguments((case["batch"], beams, vocab, keep), (s["logits"], beams * vocab, vocab), (s["scores"], beams),
                             (s["out_scores"], keep), (s["parents"], keep), (s["tokens"], keep),
                             (None, 0) if s["finished"] is None else (s["finished"], beams), s["end_token"])
        workspace = torch.empty(op.get_workspace_size(args), device="cuda", dtype=torch.uint8)
    else:
        op = ReorderStates()
        views = [state_view(src, dst, position_dim=3) for src, dst in zip(s["src"], s["dst"])]
        args = ReorderArguments((case["batch"], case["beams"], case["beams"]), (s["parents"], case["beams"]), views, s["lengths"])
    status = op.initialize(args, workspace)
    if status != Status.kSuccess:
        raise RuntimeError(f"{case}: {status!r}")
    return op


# ---- plain forms ------------------------------------------------------------------------------------------------
def _plain_q4(s):
    case = s["case"]
    w = torch.stack((s["W"] & 15, s["W"] >> 4), dim=-1).flatten(1)[:, :case["k"]].float()
    spread = torch.arange(case["k"], device="cuda") // case["group"]
    w -= 8 if s["zeros"] is None else s["zeros"].float()[:, spread]
    w *= s["scales"].float()[:, spread]
    return (s["X"].float() @ w.T).to(s["Y"].dtype)


def _plain_beam(s):
    """Order of the continuations: by their value; equal ones by the beam, then by the logit, then by the token.  The best
    of each beam are found on whole numbers that order as (logit, -token), so equal logits go to the lower token."""
    case = s["case"]
    batch, beams, vocab, keep = case["batch"], case["beams"], case["vocab"], case["keep"]
    x = s["logits"].float() + 0.0                      # one zero
    base = s["scores"].double()
    if case["normalise"]:
        top = x.amax(dim=-1, keepdim=True).double()
        top = torch.where(top.isinf(), torch.zeros_like(top), top)
        base = base - ((x.double() - top).exp().sum(dim=-1, keepdim=True).log() + top).squeeze(-1)
    bits = x.masked_fill(x.isnan(), -math.inf).view(torch.int32)
    rank = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() * 2 ** 31 - torch.arange(vocab, device="cuda")
    tokens = rank.topk(min(keep, vocab), dim=-1).indices
    value = base[..., None] + x.gather(-1, tokens).double()
    if s["finished"] is not None:                      # an ended beam goes on as it is
        done = (s["finished"] != 0)[..., None]
        alone = torch.full_like(value, -math.inf)
        alone[..., 0] = s["scores"].double()
        value = torch.where(done, alone, value)
        tokens = torch.where(done, s["end_token"], tokens)
    value = value.flatten(1)
    value = value.masked_fill(value.isnan(), -math.inf)
    value, at = value.sort(dim=-1, descending=True, stable=True)
    short = max(0, keep - value.shape[1])
    value = torch.nn.functional.pad(value[:, :keep], (0, short), value=-math.inf)
    at = torch.nn.functional.pad(at[:, :keep], (0, short))
    none = value == -math.inf
    parents = (at // min(keep, vocab)).masked_fill(none, -1).int()
    return value.float(), parents, tokens.flatten(1).gather(1, at).masked_fill(none, -1).int()


def _plain_reorder(s):
    case = s["case"]
    rows = torch.arange(case["batch"], device="cuda")[:, None]
    lengths = s["lengths"]
    if lengths is None:
        lengths = torch.full((case["batch"],), case["positions"], device="cuda")
    used = (torch.arange(case["positions"], device="cuda") < lengths[:, None])[:, None, None, :, None]
    parents = s["parents"].long()
    return [dst.copy_(torch.where(used, src[rows, parents], dst)) for src, dst in zip(s["src"], s["dst"])]


PLAIN = {"q4": _plain_q4, "beam": _plain_beam, "reorder": _plain_reorder}


def run(state):
    if not own:
        return PLAIN[state["case"]["kind"]](state)
    if state["op"].run() != 0:
        raise RuntimeError("the call was refused")
    kind = state["case"]["kind"]
    if kind == "q4":
        return state["Y"]
    if kind == "beam":
        return state["out_scores"], state["parents"], state["tokens"]
    return state["dst"]


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "q4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        return {"bytes": n * ((k + 1) // 2) + n * groups * (BYTES[case["scale"]] + case["zeros"]) + m * k * BYTES[case["x"]]
                + m * n * BYTES[case["y"]], "flops": 2 * m * n * k}
    if case["kind"] == "beam":
        rows = case["batch"] * case["beams"]
        live = rows * (0.85 if case["finished"] else 1.0)      # an ended beam's logits are not needed
        return {"bytes": live * case["vocab"] * BYTES[case["dtype"]] + rows * (4 + case["finished"])
                + case["batch"] * case["keep"] * 12, "flops": live * case["vocab"] * (3 if case["normalise"] else 1)}
    # in place, one beam of a search stays where it is in the mean
    beams = case["beams"]
    row = case["heads"] * case["dim"] * BYTES[case["dtype"]] * sum(_lengths(case)) * case["tensors"]
    return {"bytes": row * (_survivors(beams) + beams - case["in_place"]) + 4 * case["batch"] * (beams + case["ragged"]), "flops": 0}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_q4(case, s):
    n, k, group = case["n"], case["k"], case["group"]
    q = torch.empty(n, 2 * s["W"].shape[1], device="cuda", dtype=torch.float64)
    q[:, 0::2] = (s["W"] % 16).double()
    q[:, 1::2] = torch.div(s["W"], 16, rounding_mode="floor").double()
    q = q[:, :k]
    y = torch.zeros(case["m"], n, device="cuda", dtype=torch.float64)
    for j in range(-(-k // group)):
        cols = slice(j * group, min(k, (j + 1) * group))
        zero = 8.0 if s["zeros"] is None else s["zeros"][:, j:j + 1].double()
        y += (s["X"][:, cols].double() @ (q[:, cols] - zero).T) * s["scales"][:, j].double()
    return y


def _exact_beam(case, s):
    """All beams x vocab continuations in one list, sorted as they stand: equal values keep beam and token order."""
    batch, beams, vocab, keep = case["batch"], case["beams"], case["vocab"], case["keep"]
    out = torch.full((batch, keep), -math.inf, dtype=torch.float64)
    parents = torch.full((batch, keep), -1, dtype=torch.int32)
    tokens = torch.full((batch, keep), -1, dtype=torch.int32)
    for b in range(batch):
        x = s["logits"][b].double()
        if case["normalise"]:
            x = x - torch.logsumexp(x, dim=-1, keepdim=True)
        x = x + s["scores"][b].double()[:, None]
        if s["finished"] is not None:
            x[s["finished"][b] != 0] = -math.inf
            x[:, s["end_token"]] = torch.where(s["finished"][b] != 0, s["scores"][b].double(), x[:, s["end_token"]])
        x = torch.nan_to_num(x.flatten(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        value, at = torch.sort(x, descending=True, stable=True)
        value, at = value[:keep].cpu(), at[:keep].cpu()
        count = int((value > -math.inf).sum())
        out[b, :count] = value[:count]
        parents[b, :count] = (at[:count] // vocab).int()
        tokens[b, :count] = (at[:count] % vocab).int()
    return out, parents, tokens


def _exact_reorder(case, s):
    lengths, parents, out = _lengths(case), s["parents"].cpu().tolist(), []
    for src, dst in zip(s["src"], s["dst"]):
        new = dst.clone()
        for b in range(case["batch"]):
            for j in range(case["beams"]):
                new[b, j, :, :lengths[b]] = src[b, parents[b][j], :, :lengths[b]]
        out.append(new)
    return out


def exact(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = PREPARE[case["kind"]](case, g)
    return {"q4": _exact_q4, "beam": _exact_beam, "reorder": _exact_reorder}[case["kind"]](case, state)
