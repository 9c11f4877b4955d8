"""The table's gradient of attention with a relative position bias, with a table in fp32 (as models have it), against 64 bits: tolerances that a missing
piece, a zero and a coarser forward miss.

Output gradients and values are waves of the position, go_i . v_j = g(i - j): the gradient of a bucket does not cancel, so that an error relative to it
says something.  The gradient of bucket b is the sum over the pairs of b of dS = P (dP - delta), delta_i = sum_d go_id o_id.  Errors, by row i:

  u          one rounding of P: 2^-8 P where P enters its product as one bf16 value (more than 1024 tokens), 2^-16 P where as two
  delta      e_i = sum_j r_j P_j (dP_j - delta), r_j roundings of at most u (one value: the output is an average under weights that add up to 1; two: the sum is
             that of the unrounded P, and it is sum_j r_j P_j dP_j); and the output's loss is kept to 2^-16: sum_d r_d go_d o_d
  P          one value: the divisor is off by n_i = sum_j r_j P_j, which scales the row's dS
  total      the sum of all errors e_i is taken off the buckets in proportion to their share of P, m_b = sum_i P_ib / L (P_ib: the bucket's P in row i)

so that the bucket's error is sum_i e_i (P_ib - m_b) + sum_i n_i dS_ib.  The roundings are independent of each other (the scores are random) and lie evenly
within their bounds at most, with a variance of a third of the bound's square: six standard deviations.  To that come the sums in 32 bits, which may err to
one side: those of O over S = L / 16 steps of the product (twice as many with two values) and the delta's 8, (S + 8) 2^-24 of the magnitudes; dP's 8 steps,
2^-20 of them with the rounding of each; exponents of up to 32 units and exponential 2^-19, as much for the divisor; the sums of dS 2^-20 (together 2^-18)."""
import math

import pytest
import torch

from savanna_b200 import ops
from tests.test_gpu_rpe import _map

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
ONE_VALUE_FROM = 1025                    # tokens


def _waves(L):
    w = math.pi * torch.exp(-torch.arange(64, dtype=torch.float64, device=DEV) / 64 * math.log(2000.0))
    x = torch.arange(L, dtype=torch.float64, device=DEV)[:, None] * w
    return torch.stack([x.cos(), x.sin()], -1).reshape(L, 128)


def _inputs(B, L, H, nb, maxd, causal, scores=1.0, late=False):
    g = torch.Generator(device=DEV).manual_seed(L + maxd)
    qkv = scores * torch.randn(B, L, H, 384, generator=g, device=DEV)
    qkv[..., 256:] = _waves(L)[:, None]
    go = _waves(L)[:, None] * (1 + torch.arange(H, device=DEV))[:, None] / H       # heads of unequal size
    go = go.expand(B, L, H, 128).clone()
    if late:
        go[:, :L * 3 // 4] = 0
    return qkv.to(BF), torch.randn(nb, H, generator=g, device=DEV), _map(nb, maxd, causal), go.to(BF)


def _index(L, buckets, causal):
    i = torch.arange(L, device=DEV)
    d, far = i[:, None] - i[None, :], buckets.shape[0] - 1 if causal else buckets.shape[0] // 2
    return buckets.long()[d.clamp(0, far) if causal else d.clamp(-far, far) + far]


class Head:
    """One head of one sequence in 64 bits; what a row has in each bucket, [L, nb]."""

    def __init__(self, qkv, table, at, causal, go):
        self.L, self.nb, self.at = qkv.shape[0], table.shape[0], at
        q, k, self.v = (t.double() for t in qkv.split(128, dim=-1))
        self.go = go.double()
        s = q @ k.t() / math.sqrt(128) + table.double()[at]
        if causal:
            s.masked_fill_(torch.ones(self.L, self.L, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
        self.s, self.p, self.dp = s, torch.softmax(s, -1), self.go @ self.v.t()
        self.o = self.p @ self.v
        self.ds = self.p * (self.dp - (self.go * self.o).sum(-1, keepdim=True))
        self.p_rows, self.ds_rows = self.rows(self.p), self.rows(self.ds)

    def rows(self, x):
        out = torch.zeros(self.L * self.nb, dtype=torch.float64, device=DEV)
        at = torch.arange(self.L, device=DEV)[:, None] * self.nb + self.at
        return out.index_add_(0, at.reshape(-1), x.reshape(-1)).view(self.L, self.nb)

    def variance(self, share):
        """Of the bucket's error; share [nb]: m_b."""
        two = self.L < ONE_VALUE_FROM
        u = 2.0 ** -16 if two else 2.0 ** -8
        delta = (self.go * self.o).sum(-1, keepdim=True)
        e = ((self.go * self.o).square().sum(-1) * 2.0 ** -32 + (self.p * (self.dp if two else self.dp - delta)).square().sum(-1) * u ** 2) / 3
        n = 0 if two else self.p.square().sum(-1) * u ** 2 / 3
        return ((self.p_rows - share).square() * e[:, None]).sum(0) + (0 if two else (self.ds_rows.square() * n[:, None]).sum(0))

    def sums(self):
        """Of the bucket, errors of the sums in 32 bits."""
        steps = 8 + self.L / (8 if self.L < ONE_VALUE_FROM else 16)
        mag = self.go.abs() @ self.v.abs().t()
        e = steps * 2.0 ** -24 * (self.go.abs() * (self.p @ self.v.abs())).sum(-1, keepdim=True)
        return (self.rows(self.p * (e + 2.0 ** -20 * mag)) + 2.0 ** -18 * self.rows(self.ds.abs())).sum(0)

    def single(self, share):
        """The bucket's gradient of the form for more tokens: one bf16 value of P, whose sum the output is divided by; the rows' divisor gets back what the
        largest of each 64 keys lost."""
        top = self.s[:, :64].amax(-1, keepdim=True)
        e = torch.exp(self.s - top)
        w = e.to(BF).double()
        largest = torch.cat([x.amax(-1, keepdim=True) for x in e.split(64, dim=-1)], -1)
        p = e / (w.sum(-1, keepdim=True) + (largest - largest.to(BF).double()).sum(-1, keepdim=True))
        o = w @ self.v / w.sum(-1, keepdim=True)
        r = self.rows(p * (self.dp - (self.go * o).sum(-1, keepdim=True))).sum(0)
        return r - r.sum() * share


def _head(qkv, table, buckets, causal, go, h):
    """(gradient, tolerance, heads by sequence, share of P) of head h, the bias' scale apart."""
    at = _index(qkv.shape[1], buckets, causal)
    seqs = [Head(qkv[b, :, h], table[:, h], at, causal, go[b, :, h]) for b in range(qkv.shape[0])]
    share = sum(x.p_rows.sum(0) for x in seqs) / (len(seqs) * seqs[0].L)
    sums = sum(x.sums() for x in seqs)
    bound = 6 * sum(x.variance(share) for x in seqs).sqrt() + sums + share * sums.sum()
    return sum(x.ds_rows.sum(0) for x in seqs), bound, seqs, share


def _run(qkv, table, buckets, scale, causal, go):
    from savanna_b200.ops import cuda_ops
    qkv, table = qkv.clone().requires_grad_(True), table.clone().requires_grad_(True)
    o = ops.attention_rpe(qkv, table / scale, buckets, scale, causal)
    g, = torch.autograd.grad(o, table, go)
    torch.cuda.synchronize()
    cuda_ops.check_status()
    return g.double()


def _worst(err, bound):
    return float((err.abs() / (bound + 1e-30)).max())


SHAPES = [(2, 130, 64), (1, 300, 128), (3, 500, 250), (1, 777, 128), (1, 1024, 128), (2, 1025, 128), (1, 1300, 250), (2, 2048, 128), (1, 4111, 500)]


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("B,L,maxd", SHAPES)
def test_each_bucket(B, L, maxd, causal):
    nb = 32 if causal else 64
    c = _inputs(B, L, 2, nb, maxd, causal)
    got = _run(*c[:3], 4.0, causal, c[3])
    for h in range(2):
        want, bound, seqs, _ = _head(*c[:3], causal, c[3], h)
        worst = _worst(got[:, h] - want, bound)
        assert worst <= 1
        # zeros lie outside, and a gradient without the pairs of one warp: 32 queries by 32 keys next to the diagonal
        held = torch.bincount(c[2], minlength=nb) > 0
        assert bool((want.abs() > bound)[held].all())
        for i in (32, L // 2 // 128 * 128 + 64, (L - 1) // 32 * 32):
            part = torch.zeros_like(seqs[0].ds)
            part[i: i + 32, i - 32: i] = seqs[0].ds[i: i + 32, i - 32: i]
            missing = _worst(seqs[0].rows(part).sum(0), bound)
            assert missing > 1


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("L", [130, 300, 500, 777, 1023, 1024])
def test_probabilities_enter_in_two_parts(L, causal):
    """No scores but the bias, that of half the keys of a long row such that P rounds the same way everywhere: e^-0.0019 = 1 - 0.98 * 2^-9 rounds to 1.
    Gradients of the last quarter of the rows alone.  The form for more tokens would lie outside."""
    nb = 32 if causal else 64
    c = _inputs(1, L, 2, nb, L // 2, causal, scores=0.0, late=True)
    c[1].zero_()[31::32] = math.log(1 - 0.98 * 2.0 ** -9)
    got = _run(*c[:3], 1.0, causal, c[3])
    outside = 0.0
    for h in range(2):
        want, bound, seqs, share = _head(*c[:3], causal, c[3], h)
        worst = _worst(got[:, h] - want, bound)
        assert worst <= 1
        outside = max(outside, _worst(seqs[0].single(share) - want, bound))
    assert outside > 2


def test_a_long_sequence_of_many_heads():
    """More than 262144 rows times heads, whose blocks of queries come head by head; 8192 tokens a head."""
    B, L, H = 1, 8192, 33
    c = _inputs(B, L, H, 32, 128, True)
    got = _run(*c[:3], 4.0, True, c[3])
    for h in (0, 13, 32):
        want, bound, _, _ = _head(*c[:3], True, c[3], h)
        worst = _worst(got[:, h] - want, bound)
        assert worst <= 1 and bool((want.abs() > bound).sum() >= 30)


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "both"])
@pytest.mark.parametrize("L", [200, 1300, 8192])
def test_buckets_add_up_to_zero(L, causal):
    """A softmax does not change where all scores of a row grow alike, so a head's buckets add up to zero; what the roundings of delta leave of their sum
    is taken off.  Sums in 32 bits of some hundreds of distances: 2^-16 of the magnitudes."""
    g = torch.Generator(device=DEV).manual_seed(L)
    nb = 32 if causal else 64
    qkv, go = (torch.randn(1, L, 3, n, generator=g, device=DEV).to(BF) for n in (384, 128))
    table, buckets = 0.2 * torch.randn(nb, 3, generator=g, device=DEV), _map(nb, 128, causal)
    got = _run(qkv, table, buckets, 1.0, causal, go)
    assert bool((got.sum(0).abs() <= 2.0 ** -16 * got.abs().sum(0)).all())
