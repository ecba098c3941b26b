"""The decoding operators on the device against plain implementations in 64 bits."""
import math
import os
import subprocess
import sys
import threading

import pytest
import torch

from cuasr_b200 import (BeamArguments, BeamStep, DType, Q4Arguments, Q4Product, ReorderArguments, ReorderStates, Status, device_status,
                        launch_count, state_view)

pytestmark = pytest.mark.gpu
TORCH = {DType.F32: torch.float32, DType.F16: torch.float16, DType.BF16: torch.bfloat16}
REALS = list(TORCH)
INF = math.inf


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def done():
    torch.cuda.synchronize()
    assert device_status() == 0


# ---- products with 4-bit weights ----------------------------------------------------------------------------------
class Q4Case:
    def __init__(self, m, n, k, group, x=DType.BF16, y=None, scale=None, zeros=False, pad=0, byte_offset=0, seed=0):
        g = gen(seed)
        self.m, self.n, self.k, self.group = m, n, k, group
        self.types = (x, x if y is None else y, x if scale is None else scale)
        groups = -(-k // group)
        self.X = torch.randn(m, k + pad, generator=g, device="cuda").to(TORCH[x])
        row = (k + 1) // 2 + pad
        self.bytes = torch.randint(0, 256, (n * row + byte_offset,), generator=g, device="cuda", dtype=torch.uint8)
        self.W = self.bytes[byte_offset:].view(n, row)
        self.scales = ((0.5 + torch.rand(n, groups + pad, generator=g, device="cuda")) / (4 * math.sqrt(k))).to(TORCH[self.types[2]])
        # bits above the lower four of a zero point say nothing
        self.zeros = torch.randint(0, 256, (n, groups + pad), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
        self.Y = torch.full((m, n + pad), 7.0, device="cuda", dtype=TORCH[self.types[1]])

    def run(self, stream=None):
        zeros = (None, 0) if self.zeros is None else (self.zeros, self.zeros.shape[1])
        args = Q4Arguments((self.m, self.n, self.k), (self.X, self.X.shape[1]), (self.W, self.W.shape[1]),
                           (self.scales, self.scales.shape[1]), (self.Y, self.Y.shape[1]), zeros)
        assert Q4Product(*self.types, group=self.group)(args, stream=stream) == Status.kSuccess
        return self.Y[:, :self.n]

    def weights(self):
        w = torch.stack((self.W & 15, self.W >> 4), dim=-1).flatten(1)[:, :self.k].double()
        at = torch.arange(self.k, device="cuda") // self.group
        w -= 8 if self.zeros is None else (self.zeros & 15).double()[:, at]
        return w * self.scales.double()[:, at]

    def check(self):
        y, w, x = self.run(), self.weights(), self.X[:, :self.k].double()
        done()
        want = x @ w.T
        # Sums in 32 bits: every product takes part in at most min(group, k) additions inside its group, then in one per
        # group and a few that join partial sums.  A step of the tensor cores may cut off instead of rounding (2^-23 of
        # the largest term in place of 2^-24), so 2^-23 stands for each.  The result is rounded once: half an eps.
        steps = min(self.group, self.k) + -(-self.k // self.group) + 16
        bound = steps * 2.0 ** -23 * (x.abs() @ w.abs().T) + torch.finfo(y.dtype).eps / 2 * 1.001 * want.abs() + torch.finfo(y.dtype).tiny
        off = (y.double() - want).abs()
        assert (off <= bound).all(), ((off / bound).max().item(), (off > bound).sum().item())
        assert (self.Y[:, self.n:] == 7).all()


@pytest.mark.parametrize("x", REALS)
@pytest.mark.parametrize("m,n,k,group", [
    (1, 1, 1, 32), (1, 1, 2, 32), (1, 5, 31, 32), (2, 7, 33, 32), (1, 64, 64, 64), (3, 65, 129, 64), (4, 130, 256, 128), (5, 127, 257, 128),
    (7, 16, 1000, 96), (8, 100, 512, 32), (9, 33, 640, 128), (16, 200, 384, 128), (17, 48, 511, 64), (31, 72, 320, 320), (32, 128, 1024, 4096),
    (33, 96, 288, 32), (70, 40, 192, 64), (1, 1024, 4096, 128), (4, 2051, 2050, 32)])
def test_q4_matches_64_bits(cuda_device, x, m, n, k, group):
    for zeros in (False, True):
        Q4Case(m, n, k, group, x, zeros=zeros, seed=m * n + k).check()


@pytest.mark.parametrize("x", REALS)
@pytest.mark.parametrize("y", REALS)
@pytest.mark.parametrize("scale", REALS)
def test_q4_types(cuda_device, x, y, scale):
    Q4Case(3, 70, 300, 64, x, y, scale, zeros=True).check()


@pytest.mark.parametrize("pad,byte_offset", [(1, 0), (3, 1), (16, 0), (8, 16), (0, 4), (5, 8), (2, 2)])
@pytest.mark.parametrize("m", [1, 6, 20])
def test_q4_strides_and_alignments(cuda_device, m, pad, byte_offset):
    for x in (DType.F16, DType.F32):
        Q4Case(m, 150, 416, 32, x, zeros=True, pad=pad, byte_offset=byte_offset).check()


def test_q4_large_rows(cuda_device):
    Q4Case(2, 300, 20000, 128, DType.BF16, DType.F32).check()
    Q4Case(12, 20000, 640, 64, DType.F16, DType.F32, zeros=True).check()


def test_q4_extreme_activations(cuda_device):
    """Rows with infinities and NaN do not reach other rows, and large and tiny 32-bit values keep their bits."""
    c = Q4Case(4, 40, 128, 64, DType.F32)
    c.X[0] *= 1e30
    c.X[1] *= 1e-30
    c.X[2, 5] = INF
    c.X[3, 9] = math.nan
    y = c.run()
    done()
    w, x = c.weights(), c.X.double()
    for r in (0, 1):
        want = w @ x[r]
        assert ((y[r].double() - want).abs() <= 90 * 2.0 ** -23 * (w.abs() @ x[r].abs())).all()
    assert torch.equal(torch.isnan(y[2]), w[:, 5] == 0)                     # inf * 0
    assert torch.equal(y[2][w[:, 5] != 0] > 0, w[:, 5][w[:, 5] != 0] > 0)
    assert torch.isnan(y[3]).all()


def test_q4_same_bits_every_time(cuda_device):
    c = Q4Case(5, 700, 3000, 32, DType.BF16, DType.F32, zeros=True)
    first = c.run().clone()
    for _ in range(5):
        assert torch.equal(c.run(), first)
    done()


# Sizes at which the rows of weights and k are shared out in different ways: several warps to 32 rows, several blocks to k, an X
# that shared memory holds in part only, and each of them with weight rows on 16-byte boundaries and off them.
SHARED_OUT = [(1, 40, 70000, 128, DType.BF16), (1, 5000, 300, 64, DType.F16), (2, 4000, 4000, 32, DType.BF16), (3, 30000, 700, 64, DType.F32),
              (5, 64, 33000, 32, DType.F16), (8, 3000, 9000, 128, DType.F16), (10, 100, 9001, 64, DType.F32), (12, 9000, 2500, 128, DType.BF16),
              (16, 600, 14000, 64, DType.F16), (20, 17, 2049, 32, DType.BF16), (32, 64, 20000, 128, DType.BF16), (32, 5000, 4100, 128, DType.F16)]


@pytest.mark.parametrize("m,n,k,group,x", SHARED_OUT)
@pytest.mark.parametrize("byte_offset", [0, 1])
def test_q4_shared_out(cuda_device, m, n, k, group, x, byte_offset):
    Q4Case(m, n, k, group, x, DType.F32, zeros=byte_offset == 0, pad=(-(k + 1) // 2) % 16, byte_offset=byte_offset, seed=k).check()


@pytest.mark.parametrize("m,n,k,group,x", [c for c in SHARED_OUT if c[0] >= 3])
def test_q4_infinities_in_one_row(cuda_device, m, n, k, group, x):
    """An infinity, a NaN and numbers that the products do not hold, in a row each; outputs that 32 bits do not hold."""
    c = Q4Case(m, n, k, group, x, DType.F32, pad=3, seed=k)
    c.X[0, k - 1], c.X[1, 0] = -INF, math.nan
    if x != DType.F16:
        c.X[2, ::7] = 2.0 ** 40
        c.X[2, 1] = 2.0 ** 120
    y, w = c.run().clone(), c.weights()
    done()
    want = c.X[:, :k].double() @ w.T
    assert torch.isnan(y[1]).all() and torch.equal(torch.isnan(y[0]), w[:, k - 1] == 0)
    ruled = w[:, k - 1] != 0
    assert torch.equal(y[0][ruled], torch.where(w[:, k - 1] > 0, -INF, INF).float()[ruled])
    # as in Q4Case.check
    steps = min(group, k) + -(-k // group) + 16
    bound = steps * 2.0 ** -23 * (c.X[2:, :k].double().abs() @ w.abs().T) + 2.0 ** -24 * 1.001 * want[2:].abs()
    assert ((y[2:].double() - want[2:]).abs() <= bound).all()


@pytest.mark.parametrize("x", REALS)
@pytest.mark.parametrize("m,n,k,group", [(1, 70, 256, 64), (4, 300, 1000, 128), (3, 64, 4100, 8192), (11, 130, 640, 32), (20, 45, 2050, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_q4_weights_at_their_zero_points(cuda_device, x, m, n, k, group, zeros):
    """Weights that equal their zero point (padded or pruned ones) add nothing, not even a rounding, whatever the activations; few
    others among them count as in Q4Case.check, whose bound goes by |x w|."""
    for byte_offset in (0, 1):
        c = Q4Case(m, n, k, group, x, DType.F32, zeros=zeros, pad=(-(k + 1) // 2) % 16, byte_offset=byte_offset, seed=k)
        c.X += 3
        c.X[0, ::5] = 1000.25
        at = torch.arange(2 * c.W.shape[1], device="cuda").div(group, rounding_mode="floor").clamp_(max=-(-k // group) - 1)
        zero = (c.zeros & 15)[:, at] if zeros else torch.full((n, at.numel()), 8, device="cuda", dtype=torch.uint8)
        g = gen(n)

        def weigh(q):
            c.W.copy_(q[:, 0::2] | q[:, 1::2] << 4)
        weigh(zero)
        y = c.run()
        done()
        assert (c.weights() == 0).all() and torch.equal(y, torch.zeros_like(y))
        # one in 64 lies beside the zero point
        near = (torch.rand(zero.shape, generator=g, device="cuda") < 1 / 64).to(torch.uint8)
        weigh(torch.where(zero == 15, zero - near, zero + near))
        c.check()
        # a large activation on weights of zero
        c.X[:, k // 2] = 16384.0
        c.W[:, k // 4] = zero[:, k // 4 * 2] | zero[:, k // 4 * 2 + 1] << 4
        c.check()


@pytest.mark.parametrize("x", REALS)
@pytest.mark.parametrize("m", [1, 3, 10, 14])
@pytest.mark.parametrize("k,group", [(128, 128), (500, 512), (4096, 4096)])
def test_q4_one_weight_is_exact(cuda_device, x, m, k, group):
    """A weight row with one number that is not zero, scales of 1: the output is that product, rounded once.  Every bit of a 32-bit
    activation is in it."""
    n = 61
    c = Q4Case(m, n, k, group, x, DType.F32, zeros=True, seed=m)
    c.scales.fill_(1)
    c.X[:, ::3] *= 2.0 ** 10
    c.X[:, 1::3] *= 2.0 ** -10
    zero = (c.zeros & 15).expand(n, 2 * c.W.shape[1]).clone()
    at = torch.randint(0, k, (n, 1), generator=gen(k), device="cuda")
    zero.scatter_(1, at, torch.randint(0, 16, (n, 1), generator=gen(m), device="cuda", dtype=torch.uint8))
    c.W.copy_(zero[:, 0::2] | zero[:, 1::2] << 4)
    y = c.run()
    done()
    w = c.weights()
    assert ((w != 0).sum(dim=1) <= 1).all() and (w != 0).any()
    want = c.X.double()[:, at[:, 0]] * w.gather(1, at)[:, 0]      # 24 bits by four: exact in 64
    assert torch.equal(y, want.float())


def test_q4_non_finite_numbers_of_all_kinds(cuda_device):
    """Infinities and NaN reach the outputs whose weight is not zero (all, of a NaN), whichever of a NaN's bits are set; neighbouring
    rows and the largest finite numbers do not suffer."""
    c = Q4Case(8, 200, 512, 64, DType.F32, zeros=True)
    bits = c.X.view(torch.int32)
    bits[0, 3], bits[1, 4], bits[2, 5], bits[3, 6] = 0x7F800001, 0x7FFFFFFF, -1, 0x7FC00000           # NaN
    bits[4, 7], bits[5, 8] = 0x7F800000, 0x7F800000 - 2 ** 31                                         # infinities
    c.X[6, 9], c.X[7, 10:12] = 3.4e38, 2.0 ** 20
    y, w = c.run(), c.weights()
    done()
    assert torch.isnan(y[:4]).all()
    assert (torch.isnan(y[4]) == (w[:, 7] == 0)).all() and (y[4] == INF).eq(w[:, 7] > 0).all() and (y[4] == -INF).eq(w[:, 7] < 0).all()
    assert (torch.isnan(y[5]) == (w[:, 8] == 0)).all() and (y[5] == -INF).eq(w[:, 8] > 0).all() and (y[5] == INF).eq(w[:, 8] < 0).all()
    want = c.X[6:].double() @ w.T
    steps = 64 + 8 + 16                                                                               # as in Q4Case.check
    assert ((y[6:].double() - want).abs() <= steps * 2.0 ** -23 * (c.X[6:].double().abs() @ w.abs().T) + 2.0 ** -24 * 1.001 * want.abs()).all()


@pytest.mark.parametrize("x,size", [(DType.F16, 2.0 ** -22), (DType.BF16, 2.0 ** -100), (DType.F32, 2.0 ** -100)])
def test_q4_small_activations(cuda_device, x, size):
    """Subnormal half-precision activations, and ones for which 32 bits have room still, with scales that bring them back."""
    c = Q4Case(3, 50, 300, 64, x, DType.F32, DType.F32, zeros=True)
    c.X.copy_(torch.randn(3, 300, generator=gen(50), device="cuda") * size)
    c.scales *= 2.0 ** 20
    c.check()


@pytest.mark.parametrize("m,n,k,x", [(3, 40007, 700, DType.BF16), (7, 20011, 2304, DType.F16), (13, 12001, 4096, DType.BF16), (27, 20011, 4100, DType.F16),
                                     (9, 15001, 1500, DType.F32), (32, 30005, 8192, DType.F16)])
def test_q4_rounds_that_end_unevenly(cuda_device, m, n, k, x):
    """Workers with several units of weight rows, the last of which is short, and numbers of rows of X that the warps cannot share
    evenly: some lanes of a warp have an output more than others, and some of these are not finite."""
    c = Q4Case(m, n, k, 128, x, DType.F32, pad=5, seed=n)
    c.check()
    first = c.Y.clone()
    c.X[m // 2, k // 2] = math.nan
    y = c.run()
    done()
    rest = torch.arange(m, device="cuda") != m // 2
    assert torch.isnan(y[m // 2]).all() and torch.equal(y[rest], first[rest][:, :n])


def test_q4_results_beyond_a_type(cuda_device):
    """Results that 16 bits do not hold become infinite, those of all zeros are zero."""
    c = Q4Case(3, 100, 256, 64, DType.BF16, DType.F16)
    c.X[0] = 2.0 ** 17
    c.X[1] = 0
    c.W.fill_(0xFF)
    y = c.run()
    done()
    assert (y[0] == INF).all() and (y[1] == 0).all() and torch.isfinite(y[2]).all()


def test_q4_overlapping_calls_on_one_x(cuda_device):
    """Calls that share X and the weights, on two streams, each with its own Y."""
    first = Q4Case(4, 6000, 2048, 128, DType.BF16, DType.F32)
    want = first.run().clone()
    torch.cuda.synchronize()
    others = [Q4Case(4, 6000, 2048, 128, DType.BF16, DType.F32) for _ in range(2)]
    for c in others:
        c.X, c.W, c.scales = first.X, first.W, first.scales
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in others]
    for _ in range(4):
        for c, s in zip(others, streams):
            c.run(s)
    done()
    assert all(torch.equal(c.Y, want) for c in others)


# ---- beam steps -----------------------------------------------------------------------------------------------------
def plain_step(logits, scores, keep, normalise, finished, end_token):
    """Values, parents and tokens of every search on the host, sorted as documented; also a function that gives the value of
    any continuation."""
    batch, beams, vocab = logits.shape
    x = logits.double()
    base = scores.double()
    value = base[..., None] + x
    if normalise:
        value = (base - torch.logsumexp(x, dim=-1))[..., None] + x
    value = value.cpu()
    logits, scores = logits.float().cpu(), scores.cpu()
    ended = torch.zeros(batch, beams, dtype=torch.bool) if finished is None else finished.cpu() != 0
    result = []
    for s in range(batch):
        entries = []
        for b in range(beams):
            if ended[s, b]:
                entries.append((float(scores[s, b]), b, 0.0, end_token))
                continue
            row = value[s, b]
            # more than the keep best by logit cannot be among them
            order = torch.sort(torch.where(torch.isnan(logits[s, b]), -INF, logits[s, b] + 0.0), descending=True, stable=True)[1][:keep]
            entries += [(float(row[t]), b, float(logits[s, b, t]), int(t)) for t in order]
        entries = sorted((e for e in entries if e[0] > -INF), key=lambda e: (-e[0], e[1], -e[2], e[3]))[:keep]
        result.append(entries + [(-INF, -1, 0.0, -1)] * (keep - len(entries)))
    return result, value, ended


def same_choice(out, parents, tokens, want, value, ended, normalise):
    """The outputs of a step against plain_step's; returned as lists of (score, parent, token)."""
    got = [list(zip(o, p, t)) for o, p, t in zip(out.tolist(), parents.tolist(), tokens.tolist())]
    for s in range(len(got)):
        for (score, parent, token), e in zip(got[s], want[s]):
            if e[1] < 0 or e[0] == INF:
                assert (score, parent, token) == (e[0], e[1], e[3]), (s, score, parent, token, e)
                continue
            # Log-sum in mixed arithmetic: the exponential is off by 2 units of its last place (2^-22) and, through its
            # argument, by 2^-24 |d| <= 2^-24 * 1.5 * 25 for the terms that count; a thread's sum in 32
            # bits is at most 64 additions deep (16 within a tile, one per tile), the rest are 64-bit sums.  Relative to the sum that is below 2^-22 + 2^-18.7 + 2^-18; a log passes it on as
            # an absolute error.  The score is rounded once.
            slack = (2.0 ** -22 + 2.0 ** -18.7 + 2.0 ** -18) if normalise and not ended[s, e[1]] else 0.0
            assert abs(score - e[0]) <= slack + 2.0 ** -24 * abs(e[0]) * 1.001, (s, score, e)
            if (parent, token) != (e[1], e[3]):
                # only continuations of two prefixes whose values are nearer than the log-sums are exact may change places
                assert slack > 0 and parent != e[1] and abs(float(value[s, parent, token]) - e[0]) <= 2 * slack, (s, parent, token, e)
        assert len({(p, t) for _, p, t in got[s] if p >= 0}) == sum(p >= 0 for _, p, t in got[s])
    return got


def check_step(logits, scores, keep, normalise=True, finished=None, end_token=3, strides=None, alias=False, stream=None, pad=0):
    batch, beams, vocab = logits.shape
    dtype = {v: k for k, v in TORCH.items()}[logits.dtype]
    strides = strides or (logits.stride(0), logits.stride(1))
    want, value, ended = plain_step(logits, scores, keep, normalise, finished, end_token)
    old = scores.clone()
    out = torch.full((batch, keep + pad), 7.0, device="cuda")
    parents, tokens = (torch.full((batch, keep + pad), 77, device="cuda", dtype=torch.int32) for _ in range(2))
    if alias:
        out = scores
    op = BeamStep(dtype, normalise)
    args = BeamArguments((batch, beams, vocab, keep), (logits, *strides), (scores, scores.stride(0)), (out, out.stride(0)), (parents, keep + pad),
                         (tokens, keep + pad), (None, 0) if finished is None else (finished, finished.stride(0)), end_token)
    workspace = torch.full((op.get_workspace_size(args),), 255, device="cuda", dtype=torch.uint8)
    torch.cuda.synchronize()
    assert op(args, workspace, stream) == Status.kSuccess
    done()
    assert (parents[:, keep:] == 77).all() and (tokens[:, keep:] == 77).all() and (alias or (out[:, keep:] == 7).all())
    got = same_choice(out[:, :keep], parents[:, :keep], tokens[:, :keep], want, value, ended, normalise)
    assert alias or torch.equal(scores.view(torch.int32), old.view(torch.int32))
    return got


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("batch,beams,vocab,keep", [
    (1, 1, 1, 1), (1, 1, 1, 4), (2, 3, 5, 4), (3, 2, 7, 64), (1, 4, 17, 8), (2, 2, 255, 2), (1, 3, 1000, 6), (5, 7, 4099, 14), (1, 4, 32000, 8),
    (2, 5, 33333, 64), (1, 1, 131072, 1), (40, 16, 600, 32), (1, 64, 2500, 64), (300, 1, 300, 3), (1, 300, 40, 33)])
def test_beam_step_matches_64_bits(cuda_device, dtype, normalise, batch, beams, vocab, keep):
    g = gen(batch + beams + vocab)
    logits = (3 * torch.randn(batch, beams, vocab, generator=g, device="cuda")).to(TORCH[dtype])
    scores = -10 * torch.rand(batch, beams, generator=g, device="cuda")
    check_step(logits, scores, keep, normalise, pad=vocab % 3)


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("beam_pad,batch_pad,offset", [(1, 0, 0), (3, 5, 1), (0, 1, 3), (8, 16, 8), (5, 0, 7)])
def test_beam_step_strides_and_alignments(cuda_device, dtype, beam_pad, batch_pad, offset):
    batch, beams, vocab = 2, 3, 9001
    flat = torch.randn(offset + batch * (beams * (vocab + beam_pad) + batch_pad), generator=gen(5), device="cuda").to(TORCH[dtype])
    logits = flat[offset:].as_strided((batch, beams, vocab), (beams * (vocab + beam_pad) + batch_pad, vocab + beam_pad, 1), offset)
    check_step(logits, torch.zeros(batch, beams, device="cuda"), 6)


def test_beam_step_shared_logits(cuda_device):
    """One row of logits for all prefixes of all searches (strides of 0)."""
    row = torch.randn(1, 1, 5000, generator=gen(6), device="cuda")
    scores = -torch.rand(3, 4, generator=gen(7), device="cuda")
    check_step(row.expand(3, 4, 5000), scores, 8, strides=(0, 0))


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("vocab", [9, 700, 20011, 100000])
def test_beam_step_ties_go_to_the_lowest_index(cuda_device, dtype, vocab):
    scores = torch.zeros(2, 3, device="cuda")
    for logits in (torch.zeros(2, 3, vocab, device="cuda"), torch.randint(-2, 2, (2, 3, vocab), generator=gen(8), device="cuda").float(),
                   -0.0 * torch.randint(0, 2, (2, 3, vocab), generator=gen(9), device="cuda").float()):
        got = check_step(logits.to(TORCH[dtype]), scores, 8, normalise=False)
        assert all(s[0][1] == 0 for s in got)


@pytest.mark.parametrize("vocab", [5000, 90000])
def test_beam_step_orders_that_fill_the_lists(cuda_device, vocab):
    """Logits that rise along the vocabulary replace all candidates again and again; falling ones keep the first."""
    rising = torch.arange(vocab, device="cuda").float().div(vocab).expand(1, 2, vocab).contiguous()
    scores = torch.tensor([[0.0, -0.5 / vocab]], device="cuda")
    for keep in (1, 16, 64):
        check_step(rising, scores, keep, normalise=False)
        check_step(rising.flip(-1).contiguous(), scores, keep, normalise=False)


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("normalise", [False, True])
def test_beam_step_masks(cuda_device, dtype, normalise):
    """Half of the tokens, all but two, all of one prefix, and all of a search ruled out; the type's lowest value is a value."""
    g = gen(10)
    logits = torch.randn(4, 3, 12345, generator=g, device="cuda").to(TORCH[dtype])
    logits[0].masked_fill_(torch.rand(12345, generator=g, device="cuda") < 0.5, -INF)
    logits[1, :, 2:] = -INF
    logits[2, 1] = -INF
    logits[3] = -INF
    scores = -torch.rand(4, 3, generator=g, device="cuda")
    got = check_step(logits, scores, 7, normalise)
    assert all(e == (-INF, -1, -1) for e in got[3]) and sum(e[1] >= 0 for e in got[1]) == 6 and all(e[1] != 1 for e in got[2])
    lowest = torch.full((1, 2, 900), torch.finfo(TORCH[dtype]).min, device="cuda", dtype=TORCH[dtype])
    lowest[0, 0, 500] = 1.0
    got = check_step(lowest, torch.zeros(1, 2, device="cuda"), 5, normalise)
    assert all(e[1] >= 0 for e in got[0])


@pytest.mark.parametrize("normalise", [False, True])
def test_beam_step_infinities_and_nan(cuda_device, normalise):
    logits = torch.randn(3, 4, 3000, generator=gen(11), device="cuda")
    scores = torch.tensor([[0.0, -INF, math.nan, -1.0], [INF, 0.0, -1.0, -2.0], [0.0, -1.0, -2.0, -3.0]], device="cuda")
    logits[2, 0, 17] = math.nan
    logits[2, 1, 18] = INF
    logits[2, 2, 19] = -INF
    got = check_step(logits, scores, 9, normalise)
    assert {e[1] for e in got[0]} <= {0, 3} and {e[1] for e in got[1]} == {0}
    assert all((e[1], e[2]) != (0, 17) for e in got[2])
    if normalise:
        assert {e[1] for e in got[2]} <= {2, 3}
    else:
        assert got[2][0] == (INF, 1, 18)


@pytest.mark.parametrize("normalise", [False, True])
def test_beam_step_finished_prefixes(cuda_device, normalise):
    g = gen(12)
    logits = torch.randn(4, 5, 2222, generator=g, device="cuda")
    scores = -3 * torch.rand(4, 5, generator=g, device="cuda")
    finished = torch.zeros(4, 5, device="cuda", dtype=torch.uint8)
    finished[0, 2] = 1
    finished[1, :4] = 255
    finished[2] = 1
    scores[2, 3] = -INF
    logits[0, 2] = math.nan               # not looked at
    got = check_step(logits, scores, 6, normalise, finished, end_token=2000000000)
    assert [e[2] for e in got[2]] == [2000000000] * 4 + [-1] * 2
    wide = torch.zeros(4, 9, device="cuda", dtype=torch.uint8)
    wide[:, :5] = finished
    check_step(logits, scores, 6, normalise, wide[:, :5])


def test_beam_step_first_step_and_scores_in_place(cuda_device):
    logits = torch.randn(3, 4, 1500, generator=gen(13), device="cuda", dtype=torch.float32)
    scores = torch.full((3, 4), -INF, device="cuda")
    scores[:, 0] = 0.0
    got = check_step(logits, scores, 4, alias=True)
    assert all(e[1] == 0 for s in got for e in s)


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("vocab", [4000, 131071])
@pytest.mark.parametrize("keep", [1, 33, 64])
def test_beam_step_runs_of_equal_logits(cuda_device, dtype, vocab, keep):
    """Plateaus that rise along the vocabulary, each wider than a warp's room for candidates, and one that begins inside another
    tile than it ends; equal values between prefixes too."""
    steps = torch.arange(vocab, device="cuda") // 700
    logits = torch.stack((steps, steps.flip(0), steps % 3)).float().to(TORCH[dtype])[None].contiguous()
    check_step(logits, torch.zeros(1, 3, device="cuda"), keep, normalise=False)


@pytest.mark.parametrize("normalise", [False, True])
@pytest.mark.parametrize("beams,keep", [(257, 4), (1024, 8), (130, 64), (512, 17)])
def test_beam_step_many_prefixes(cuda_device, normalise, beams, keep):
    g = gen(beams)
    logits = torch.randint(-3, 4, (2, beams, 50), generator=g, device="cuda").float()
    finished = (torch.rand(2, beams, generator=g, device="cuda") < 0.3).to(torch.uint8)
    scores = -torch.randint(0, 3, (2, beams), generator=g, device="cuda").float()
    scores[1, ::2] = -INF
    check_step(logits + torch.rand(2, beams, 50, generator=g, device="cuda") * normalise, scores, keep, normalise, finished)


@pytest.mark.parametrize("normalise", [False, True])
def test_beam_step_bound_at_the_end_of_a_row(cuda_device, normalise):
    """Rows of three tiles whose eighth best is the second best of one warp, which holds the smallest bound and a maximum far above
    it: every warp has to take that bound, however far the others are.  Each of 1024 rows, again and again."""
    rows, lanes, tile = 1024, 128, 2048
    x = torch.randn(rows, 3 * tile, generator=gen(40), device="cuda").clamp_(-2, 2) - 8
    for poor in range(4):
        for warp in range(4):
            high = (6.5, 1.0) if warp == poor else (5.0 + warp / 8, 5.5 + warp / 8)
            for lane, value in zip((32 * warp + poor, 32 * warp + 31 - poor), high):
                x[poor::4, tile * (lane % 3) + lane * 4 + poor] = value
    scores = torch.zeros(64, 16, device="cuda")
    keep = 8
    value, token = x.topk(keep, dim=1)
    # the searches' best are among their prefixes' best, equal values of the lower prefix
    at = value.view(64, -1).sort(dim=1, descending=True, stable=True)[1][:, :keep]
    want = (at // keep).int(), token.view(64, -1).gather(1, at).int()
    # searches of one prefix, too, whose outputs are all that the prefix has
    for batch, beams in ((rows, 1),) if normalise else ((64, 16), (rows, 1)):
        out = torch.empty(batch, keep, device="cuda")
        parents, tokens = (torch.empty(batch, keep, device="cuda", dtype=torch.int32) for _ in range(2))
        op = BeamStep(DType.F32, normalise)
        args = BeamArguments((batch, beams, 3 * tile, keep), (x, beams * 3 * tile, 3 * tile), (scores, beams), (out, keep), (parents, keep), (tokens, keep))
        workspace = torch.empty(op.get_workspace_size(args), device="cuda", dtype=torch.uint8)
        assert op.initialize(args, workspace) == Status.kSuccess
        wrong = torch.zeros((), device="cuda", dtype=torch.int64)
        for _ in range(200):
            assert op.run(torch.cuda.current_stream()) == Status.kSuccess
            wrong += (tokens != (token if beams == 1 else want[1])).sum() + (parents != (0 if beams == 1 else want[0])).sum()
        done()
        assert wrong.item() == 0


@pytest.mark.parametrize("dtype", REALS)
@pytest.mark.parametrize("shape", ["flat", "rising"])
def test_beam_step_log_sums_of_long_rows(cuda_device, dtype, shape):
    """1040 prefixes, so that a block has a whole row, of 2^23 logits: small terms that a sum in 32 bits would not notice one by one but
    that count together, and logits that rise a little from tile to tile.  All prefixes have the one row (strides of 0)."""
    batch, beams, vocab, keep = 65, 16, 2 ** 23, 2
    if shape == "flat":
        row = torch.full((vocab,), -16.7, device="cuda")
        row[:4096] = 0
    else:
        row = torch.arange(vocab, device="cuda", dtype=torch.float64).mul_(20 / vocab).float()
    row = row.to(TORCH[dtype])
    scores = torch.zeros(batch, beams, device="cuda")
    out = torch.empty(batch, keep, device="cuda")
    parents, tokens = (torch.empty(batch, keep, device="cuda", dtype=torch.int32) for _ in range(2))
    op = BeamStep(dtype)
    args = BeamArguments((batch, beams, vocab, keep), (row, 0, 0), (scores, beams), (out, keep), (parents, keep), (tokens, keep))
    assert op(args, torch.empty(op.get_workspace_size(args), device="cuda", dtype=torch.uint8)) == Status.kSuccess
    done()
    want = (row.double().max() - torch.logsumexp(row.double(), dim=0)).item()
    # The exponentials and their arguments as in same_choice (the terms lie within 25 of the reference, which a thread's maximum may pass by
    # 16), twice where the reference is taken anew or the threads' meet, and a tile's sum of up to 32 in 32 bits, ten additions deep; the
    # score is rounded once.
    slack = 3 * (2.0 ** -22 + 2.0 ** -18.7) + 10 * 2.0 ** -24
    assert (out.double() - want).abs().max().item() <= slack + 2.0 ** -24 * 1.001 * abs(want)
    best = torch.nonzero(row == row.max())[:keep, 0]
    if best.numel() == keep:
        assert (parents == 0).all() and (tokens == best.int()).all()


def test_beam_step_logits_beyond_32_bit_offsets(cuda_device):
    """Element offsets above 2^31: two searches whose rows lie 2^31 + 16 half-precision numbers apart."""
    far = 2 ** 31 + 16
    flat = torch.empty(far + 5000, device="cuda", dtype=torch.float16)
    flat[:5000] = torch.randn(5000, generator=gen(14), device="cuda")
    flat[far:] = torch.randn(5000, generator=gen(15), device="cuda")
    check_step(flat.as_strided((2, 1, 5000), (far, 5000, 1)), torch.zeros(2, 1, device="cuda"), 5)


# ---- reordering ------------------------------------------------------------------------------------------------------
def check_reorder(src, parents, dst=None, lengths=None, position_dim=None, stream=None):
    """src, dst: lists of tensors; dst None: in place."""
    views = [state_view(s, None if dst is None else d, position_dim) for s, d in zip(src, dst or src)]
    batch, keep = parents.shape
    beams = src[0].shape[1]
    before = [d.clone() for d in (dst or src)]
    want = [b.clone() for b in before]
    for old, new, s in zip(before, want, src if dst else before):
        for b in range(batch):
            for j, p in enumerate(parents[b].tolist()):
                if 0 <= p < beams:
                    row = s[b, p]
                    if lengths is None or position_dim is None:
                        new[b, j] = row
                    else:
                        n = min(max(int(lengths[b]), 0), src[0].shape[position_dim])
                        new[b, j].narrow(position_dim - 2, 0, n).copy_(row.narrow(position_dim - 2, 0, n))
    args = ReorderArguments((batch, beams, keep), (parents, parents.stride(0)), views, lengths)
    torch.cuda.synchronize()
    assert ReorderStates()(args, stream=stream) == Status.kSuccess
    torch.cuda.synchronize()
    for got, w in zip(dst or src, want):
        assert torch.equal(got, w)


def parents_of(batch, beams, keep, seed, low=0):
    return torch.randint(low, beams, (batch, keep), generator=gen(seed), device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("batch,beams,keep", [(1, 1, 1), (1, 4, 4), (3, 5, 5), (2, 8, 3), (2, 9, 9), (1, 16, 16), (2, 17, 17), (1, 32, 32), (4, 40, 20)])
def test_reorder_rows(cuda_device, in_place, batch, beams, keep):
    g = gen(batch * beams)
    src = [torch.randn(batch, beams, *shape, generator=g, device="cuda").to(t)
           for shape, t in (((3, 7, 8), torch.bfloat16), ((1000,), torch.float32), ((5,), torch.float64), ((), torch.int32))]
    dst = None if in_place else [torch.zeros(batch, keep, *s.shape[2:], device="cuda", dtype=s.dtype) for s in src]
    check_reorder(src, parents_of(batch, beams, keep, beams, low=-1), dst)
    done()


def test_reorder_cycles_in_place(cuda_device):
    x = torch.randn(3, 6, 5000, generator=gen(1), device="cuda")
    check_reorder([x], torch.tensor([[1, 2, 3, 4, 5, 0], [5, 4, 3, 2, 1, 0], [0, 1, 2, 3, 4, 5]], device="cuda", dtype=torch.int32))
    done()


def test_reorder_into_more_rows(cuda_device):
    src = [torch.randn(2, 3, 500, generator=gen(2), device="cuda")]
    for keep in (5, 33, 70):
        check_reorder(src, parents_of(2, 3, keep, keep), [torch.zeros(2, keep, 500, device="cuda")])
    done()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("order", ["heads", "positions", "outermost", "cut"])
def test_reorder_padded_caches(cuda_device, in_place, order):
    """Positions behind a search's length stay as they were, whatever the order of the dimensions; lengths of 0, 1, all, and
    outside of the range."""
    batch, beams, heads, positions, dim = 6, 4, 3, 37, 24
    def make(seed):
        x = torch.randn(2 * batch * beams * heads * positions * dim, generator=gen(seed), device="cuda").to(torch.bfloat16)
        if order == "heads":
            return x[:x.numel() // 2].view(batch, beams, heads, positions, dim), 3
        if order == "positions":
            return x[:x.numel() // 2].view(batch, beams, positions, heads, dim), 2
        if order == "outermost":
            return x[:x.numel() // 2].view(positions, batch, beams, heads * dim).permute(1, 2, 0, 3), 2
        return x.view(batch, beams, heads, 2 * positions, dim)[:, :, :, :positions], 3
    lengths = torch.tensor([0, 1, 20, positions, -5, 1000], device="cuda", dtype=torch.int32)
    src = [make(seed)[0] for seed in (3, 4)]
    dst = None if in_place else [make(seed)[0] for seed in (5, 6)]
    check_reorder(src, parents_of(batch, beams, beams, 7), dst, lengths, make(0)[1])
    check_reorder(src, parents_of(batch, beams, beams, 8), dst, None, make(0)[1])
    done()


@pytest.mark.parametrize("size", [1, 2, 3, 6, 8, 12, 15, 16, 17, 48, 1001])
@pytest.mark.parametrize("offset", [0, 1, 2, 4, 8])
def test_reorder_alignments(cuda_device, size, offset):
    flat = torch.randint(0, 256, (offset + 2 * 3 * 5 * size,), generator=gen(size), device="cuda", dtype=torch.uint8)
    x = flat[offset:].view(2, 3, 5, size)
    check_reorder([x], parents_of(2, 3, 3, size))
    check_reorder([x], parents_of(2, 3, 3, size + 1), None, torch.tensor([2, 4], device="cuda", dtype=torch.int32), 2)
    done()


def test_reorder_many_states(cuda_device):
    src = [torch.randn(2, 3, 4, 1 + i % 7, generator=gen(i), device="cuda") for i in range(150)]
    before = launch_count()
    check_reorder(src, parents_of(2, 3, 3, 1))
    assert launch_count() - before == 3                       # 64 states to a launch
    done()


def test_reorder_does_not_follow_parents_out_of_range(cuda_device):
    x = torch.randn(2, 3, 100, generator=gen(9), device="cuda")
    check_reorder([x], torch.tensor([[2, 3, 0], [0, 2 ** 31 - 1, -2 ** 31]], device="cuda", dtype=torch.int32))
    assert device_status() == 4 and device_status() == 0


def test_reorder_ignores_lengths_out_of_range(cuda_device):
    x = torch.randn(3, 4, 2, 11, 8, generator=gen(31), device="cuda")
    lengths = torch.tensor([-5, 2 ** 31 - 1, 0], device="cuda", dtype=torch.int32)
    check_reorder([x], parents_of(3, 4, 4, 32), lengths=lengths, position_dim=3)
    done()


def test_reorder_of_a_cache_without_positions_yet(cuda_device):
    """As at the first step of a search: the cache has no positions in use, the other states move."""
    cache = torch.randn(2, 3, 4, 10, 8, generator=gen(33), device="cuda")
    old, x, parents = cache.clone(), torch.randn(2, 3, 50, generator=gen(34), device="cuda"), parents_of(2, 3, 3, 35)
    want = x.gather(1, parents.long()[..., None].expand(-1, -1, 50))
    args = ReorderArguments((2, 3, 3), (parents, 3), [state_view(cache[:, :, :, :0], position_dim=3), state_view(x), state_view(cache[:, :, :0])])
    before = launch_count()
    assert ReorderStates()(args) == Status.kSuccess
    done()
    assert torch.equal(x, want) and torch.equal(cache, old) and launch_count() - before == 1


def test_reorder_beyond_32_bit_offsets(cuda_device):
    """Beams that lie more than 2^32 bytes apart."""
    far = 2 ** 32 + 64
    flat = torch.zeros(far + 1024, device="cuda", dtype=torch.uint8)
    x = flat.as_strided((1, 2, 1024), (0, far, 1))
    x[0, 0], x[0, 1] = 3, 5
    x[0, 1, 700:] = 9
    check_reorder([x], torch.tensor([[1, 0]], device="cuda", dtype=torch.int32))
    done()


# ---- the operators together --------------------------------------------------------------------------------------------
class Decoder:
    """A loop as a program has it: hidden rows -> logits -> step -> states and hidden rows follow the beams."""

    def __init__(self, seed, batch=2, beams=4, hidden=256, vocab=5003):
        g = gen(seed)
        self.batch, self.beams, self.vocab = batch, beams, vocab
        self.q4 = Q4Case(batch * beams, vocab, hidden, 64, DType.BF16, DType.F32, zeros=True, seed=seed)
        self.scores = torch.full((batch, beams), -INF, device="cuda")
        self.scores[:, 0] = 0
        self.finished = torch.zeros(batch, beams, device="cuda", dtype=torch.uint8)
        self.parents, self.tokens = (torch.zeros(batch, beams, device="cuda", dtype=torch.int32) for _ in range(2))
        self.cache = torch.randn(batch, beams, 2, 9, 16, generator=g, device="cuda").to(torch.bfloat16)
        self.hidden = self.q4.X.view(batch, beams, hidden)
        self.lengths = torch.tensor([9, 4], device="cuda", dtype=torch.int32)
        c = self.q4
        self.product, self.step, self.reorder = Q4Product(*c.types, group=64), BeamStep(DType.F32), ReorderStates()
        logits, rows = c.Y, (batch, beams)
        step_args = BeamArguments((*rows, vocab, beams), (logits, beams * vocab, vocab), (self.scores, beams), (self.scores, beams),
                                  (self.parents, beams), (self.tokens, beams), (self.finished, beams))
        self.workspace = torch.empty(self.step.get_workspace_size(step_args), device="cuda", dtype=torch.uint8)
        assert self.product.initialize(Q4Arguments((batch * beams, vocab, hidden), (c.X, hidden), (c.W, c.W.shape[1]),
                                                   (c.scales, c.scales.shape[1]), (logits, vocab), (c.zeros, c.zeros.shape[1]))) == 0
        assert self.step.initialize(step_args, self.workspace) == 0
        assert self.reorder.initialize(ReorderArguments((*rows, beams), (self.parents, beams),
                                                        [state_view(self.cache, position_dim=3), state_view(self.hidden)], self.lengths)) == 0

    def enqueue(self, stream=None):
        handle = torch.cuda.current_stream() if stream is None else stream
        for op in (self.product, self.step, self.reorder):
            assert op.run(handle) == Status.kSuccess

    def state(self):
        return [t.clone() for t in (self.q4.Y, self.scores, self.parents, self.tokens, self.cache, self.hidden)]


def test_operators_together(cuda_device):
    """Every operator's result from what the one before it left.  (Prefixes of one parent have the same hidden rows here, so
    their continuations a b and b a have equal values but for roundings: same_choice allows either.)"""
    d = Decoder(21)
    rows = torch.arange(d.batch, device="cuda")[:, None]
    used = (torch.arange(9, device="cuda") < d.lengths[:, None])[:, None, None, :, None]
    for _ in range(4):
        _, scores, _, _, cache, hidden = d.state()
        d.enqueue()
        done()
        w, x = d.q4.weights(), hidden.view(-1, hidden.shape[-1]).double()
        assert ((d.q4.Y.double() - x @ w.T).abs() <= 90 * 2.0 ** -23 * (x.abs() @ w.abs().T)).all()
        want = plain_step(d.q4.Y.view(d.batch, d.beams, d.vocab), scores, d.beams, True, d.finished, 0)
        same_choice(d.scores, d.parents, d.tokens, *want, True)
        parents = d.parents.long()
        assert torch.equal(d.cache, torch.where(used, cache[rows, parents], cache)) and torch.equal(d.hidden, hidden[rows, parents])


def test_a_search_whose_prefixes_end(cuda_device):
    """The flags of ended prefixes follow the back-pointers like the other states, and the tokens set them: as in README.md."""
    batch, beams, vocab, end = 3, 4, 300, 7
    g = gen(41)
    table = 2 * torch.randn(batch, vocab, vocab, generator=g, device="cuda")          # logits by the token before
    table[:, :, end] += 2.0
    logits = torch.empty(batch, beams, vocab, device="cuda")
    scores = torch.full((batch, beams), -INF, device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros(batch, beams, device="cuda", dtype=torch.uint8)
    parents, tokens = (torch.zeros(batch, beams, device="cuda", dtype=torch.int32) for _ in range(2))
    texts = torch.full((batch, beams, 64), -1, device="cuda", dtype=torch.int32)
    step, reorder, rows = BeamStep(DType.F32), ReorderStates(), torch.arange(batch, device="cuda")[:, None]
    args = BeamArguments((batch, beams, vocab, beams), (logits, beams * vocab, vocab), (scores, beams), (scores, beams), (parents, beams),
                         (tokens, beams), (finished, beams), end)
    workspace = torch.empty(step.get_workspace_size(args), device="cuda", dtype=torch.uint8)
    assert step.initialize(args, workspace) == Status.kSuccess
    assert reorder.initialize(ReorderArguments((batch, beams, beams), (parents, beams), [state_view(finished), state_view(texts)])) == Status.kSuccess
    stream, before = torch.cuda.current_stream(), torch.zeros(batch, beams, device="cuda", dtype=torch.int64)
    for i in range(64):
        logits.copy_(table[rows, before])
        old_scores, old_finished, old_texts = scores.clone(), finished.clone(), texts.clone()
        want = plain_step(logits, old_scores, beams, True, old_finished, end)
        for op in (step, reorder):
            assert op.run(stream) == Status.kSuccess
        done()
        same_choice(scores, parents, tokens, *want, True)
        assert torch.equal(finished, old_finished[rows, parents.long()]) and torch.equal(texts, old_texts[rows, parents.long()])
        assert (tokens[finished != 0] == end).all()
        assert torch.equal(scores[finished != 0], old_scores[rows, parents.long()][finished != 0])
        texts[:, :, i] = tokens
        finished.logical_or_(tokens == end)
        before = tokens.long()
    assert finished.any(dim=1).all()
    # what follows the end of a prefix is the end again
    ended_at = (texts == end).int().argmax(dim=2)
    behind = torch.arange(64, device="cuda") >= ended_at[..., None]
    assert (texts[behind & (finished != 0)[..., None]] == end).all()


def test_captured_steps_replay_like_eager_ones(cuda_device):
    eager, captured = Decoder(22), Decoder(22)
    for _ in range(3):
        eager.enqueue()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured.enqueue()
    for _ in range(3):
        graph.replay()
    done()
    for a, b in zip(eager.state(), captured.state()):
        assert torch.equal(a, b)


def test_two_searches_on_two_streams(cuda_device):
    alone = [Decoder(seed, vocab=20011) for seed in (23, 24)]
    both = [Decoder(seed, vocab=20011) for seed in (23, 24)]
    for d in alone:
        for _ in range(5):
            d.enqueue()
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in both]
    for _ in range(5):
        for d, s in zip(both, streams):
            d.enqueue(s)
    done()
    for d, e in zip(alone, both):
        for a, b in zip(d.state(), e.state()):
            assert torch.equal(a, b)


def test_the_first_calls_of_a_process_can_be_captured(cuda_device):
    """In a process of its own: nothing is looked up on the device before the capture."""
    code = """
import sys
sys.path.insert(0, "tests")
import torch
from test_decode_gpu import Decoder
d, e = Decoder(25, vocab=20011), Decoder(25, vocab=20011)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    d.enqueue()
for _ in range(2):
    graph.replay()
    e.enqueue()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(d.state(), e.state()))
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_calls_from_two_threads(cuda_device):
    alone, both = [Decoder(seed) for seed in (26, 27)], [Decoder(seed) for seed in (26, 27)]
    for d in alone:
        for _ in range(20):
            d.enqueue()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in both]
    threads = [threading.Thread(target=lambda d=d, s=s: [d.enqueue(s) for _ in range(20)]) for d, s in zip(both, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    done()
    for d, e in zip(alone, both):
        for a, b in zip(d.state(), e.state()):
            assert torch.equal(a, b)


def test_replays_of_two_graphs_that_share_a_workspace(cuda_device):
    """One after the other on one stream: the workspace is overwritten by every step."""
    a, b, alone = Decoder(28), Decoder(29), [Decoder(28), Decoder(29)]
    b.workspace = a.workspace
    rows, vocab = (b.batch, b.beams), b.vocab
    args = BeamArguments((*rows, vocab, b.beams), (b.q4.Y, b.beams * vocab, vocab), (b.scores, b.beams), (b.scores, b.beams),
                         (b.parents, b.beams), (b.tokens, b.beams), (b.finished, b.beams))
    assert b.step.initialize(args, a.workspace) == 0
    graphs = []
    for d in (a, b):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            d.enqueue()
    for _ in range(3):
        for g in graphs:
            g.replay()
    for d in alone:
        for _ in range(3):
            d.enqueue()
    done()
    for d, e in zip((a, b), alone):
        for x, y in zip(d.state(), e.state()):
            assert torch.equal(x, y)
