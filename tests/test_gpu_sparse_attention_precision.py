"""sparse_attention held to the roundings that it makes, and no others: q is not rounded with the scale in it, so a score is off by the fp32 sums alone.

Worst case, per element.  A = max_j sum_i |q_i k_ji| scale; p: the exact weights; mag = sum_j p_j |v_j|; n keys.
  scores    128 products and the row's reference summed in fp32, each addition off by at most 2^-23 of the running magnitude (the matrix instruction may truncate), which is at
            most 2 A; the scaling's two roundings: eps = (128 + 8) 2^-23 2 A, a weight off by a factor e^eps, numerator and row sum
  weights   rounded to bf16 (2^-8) in front of the product with v.  The kernel for more than 16 queries sums the rounded weights, the other the unrounded ones: 2^-8 (mag + |o|) and 2^-8 mag
  sums      n + 200 additions, numerator and row sum, 2^-23 each; exp2, rescaling, division: within the 200
  output    2^-8 |o|
Together, for random inputs: the errors of weights and of outputs are independent and each uniform within half a step, at most 2^-8 / sqrt(3) of the value in the root mean square; v
independent of the weights with mean 0 makes sum_j p_j^2 (v_j - o)^2 and o^2 the same in the mean, so the whole output is off by at most sqrt(2 / 3) 2^-8 of its norm, 0.0032 (about
0.0023 where mantissas are spread evenly).  With scores of spread 4 a q that had been rounded with its scale would be off by 4 times 0.0016 in the exponent alone."""
import math

import pytest
import torch

from test_gpu_sparse_attention import BF, F64, SCALE, SHAPES, lens_of, lists, rnd, vt_of
from test_gpu_sparse_attention import gen, ops  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu
RMS = math.sqrt(2 / 3) * 2.0 ** -8


def exact(q, k, vt, index, count=None, lens=None, scale=SCALE):
    """(o, bound of an element's error) in 64 bits, the bound without the output's rounding of what lies within it"""
    B, Lq, H, D = q.shape
    Bk, Lk, Hk, _ = k.shape
    o = torch.zeros(B, Lq, H, D, dtype=F64, device=q.device)
    bound = torch.zeros_like(o)
    entries = index.cpu()
    for b in range(B):
        end = Lk if lens is None else min(max(int(lens[b % Bk]), 0), Lk)
        for h in range(H):
            hk = h // (H // Hk)
            kh, vh = k[b % Bk, :, hk].to(F64), vt[b % Bk, hk * 128 : hk * 128 + 128, :Lk].to(F64).t()
            for n in range(entries.shape[2]):
                c = entries.shape[3] if count is None else min(max(int(count[b, h, n]), 0), entries.shape[3])
                keys = [j for e in entries[b, h, n, :c].tolist() if e >= 0 for j in range(min(64 * e, end), min(64 * e + 64, end))]
                if not keys:
                    continue
                at = torch.tensor(keys, device=q.device)
                rows = slice(128 * n, 128 * n + 128)
                qq = q[b, rows, h].to(F64)
                p = torch.softmax(qq @ kh[at].t() * scale, 1)
                A = (qq.abs() @ kh[at].abs().t() * scale).amax(1, keepdim=True)
                r, mag = p @ vh[at], p @ vh[at].abs()
                eps = 136 * 2.0 ** -23 * 2 * A
                both = mag + r.abs()
                weights = 2.0 ** -8 * (both if Lq > 16 else mag)
                o[b, rows, h] = r
                bound[b, rows, h] = 1.02 * (weights + torch.expm1(eps) * both + 2 * (len(keys) + 200) * 2.0 ** -23 * mag)
    return o, bound + 2.0 ** -8 * (o.abs() + bound)


def held(got, o, bound, rms=True):
    d = got.to(F64) - o
    assert torch.isfinite(d).all()
    assert (d.abs() <= bound + 1e-30).all(), (d.abs() / (bound + 1e-30)).max().item()
    if rms:
        assert d.norm() <= RMS * o.norm(), (d.norm() / o.norm()).item()


@pytest.mark.parametrize("B,Bk,H,Hk,Lq,Lk,keep,lens", SHAPES + [(1, 1, 30, 1, 2300, 5000, 70, None), (2, 1, 20, 20, 1665, 640, 4, [577]), (1, 1, 1, 1, 17, 4000, 60, None), (1, 1, 12, 12, 1560, 4096, 48, [4001])])
@pytest.mark.parametrize("gain", [1.0, 4.0])
@pytest.mark.parametrize("prescaled", [False, True])
def test_within_its_roundings(ops, B, Bk, H, Hk, Lq, Lk, keep, lens, gain, prescaled):
    g = gen(Lq + 3 * Lk)
    q, k, v = rnd(g, B, Lq, H, 128, gain=gain), rnd(g, Bk, Lk, Hk, 128), rnd(g, Bk, Lk, Hk, 128)
    if prescaled:
        q = (q.float() * ops.attention_qscale()).to(BF)
    index = lists(g, B, H, (Lq + 127) // 128, (Lk + 63) // 64, keep)
    vt = vt_of(v)
    got = ops.sparse_attention(q, k, vt, index, k_lens=lens_of(lens), q_prescaled=prescaled)
    held(got, *exact(q, k, vt, index, None, lens, math.log(2.0) if prescaled else SCALE))
    assert torch.equal(got, ops.sparse_attention(q, k, vt, index, k_lens=lens_of(lens), q_prescaled=prescaled))


@pytest.mark.parametrize("Lq", [9, 130, 700])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("step", [2, 30])
def test_maxima_that_rise_or_fall_along_the_list(ops, Lq, sign, step):
    """Scores that climb (or fall) by `step` powers of e or more from block to block: the running reference follows them late or every time, and what was summed before has to
    be scaled down exactly.  A lost or doubled rescaling changes outputs by their own size, which the bound stays far below: with 64 to 90 keys of about the same weight the
    largest |o| is some 3 / sqrt(90) = 0.3, the bound 2^-8 (0.8 + 2 * 0.3) + 0.0086 * (0.8 + 0.3) = 0.015 (scores up to 300: eps = 136 * 2^-23 * 600 * 0.7 = 0.007 and the sums)."""
    g = gen(Lq + step)
    blocks = 20 if step == 30 else 150
    L = 64 * blocks
    k = rnd(g, 1, L, 1, 128, gain=0.02)
    k[0, :, 0, 0] += (torch.arange(L, device="cuda") // 64 * (step / 8) * sign).to(BF)
    q = rnd(g, 1, Lq, 1, 128, gain=0.1)
    q[0, :, 0, 0] = 8.0
    q[0, ::3, 0, 0] = -8.0
    v = rnd(g, 1, L, 1, 128)
    index = torch.arange(blocks, dtype=torch.int32, device="cuda").expand(1, 1, (Lq + 127) // 128, blocks).contiguous()
    vt = vt_of(v)
    got = ops.sparse_attention(q, k, vt, index, q_prescaled=True)
    o, bound = exact(q, k, vt, index, scale=math.log(2.0))
    assert bound.max() < o.abs().max() / 8, (bound.max().item(), o.abs().max().item())   # (the oracle alone: whether the test can see anything)
    held(got, o, bound, rms=False)


NANS = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("H,keep", [(2, 6), (1, 40), (520, 3)])
@pytest.mark.parametrize("what", NANS)
def test_a_value_that_is_no_number_shows_where_it_is_attended(ops, H, keep, what):
    """In a key or a query: every output of the rows that attend it is NaN (an infinite score against a finite one is); the other rows, of other lists and other heads, are what they
    are without it.  Whole lists, lists in shares, more lists than run at a time."""
    g = gen(H + keep)
    Lq, Lk = 260, 64 * (2 * keep + 1) - 10
    q, k, v = rnd(g, 1, Lq, H, 128), rnd(g, 1, Lk, H, 128), rnd(g, 1, Lk, H, 128)
    nk = (Lk + 63) // 64
    index = torch.stack([torch.arange(keep), torch.arange(keep, 2 * keep), torch.tensor([nk - 1] * keep)]).to(torch.int32).expand(1, H, 3, keep).contiguous().cuda()
    vt = vt_of(v)
    clean = ops.sparse_attention(q, k, vt, index)
    for block in (0, keep - 1, keep // 2):                                # first, last, in the middle of the first list
        bad = k.clone()
        bad[0, 64 * block + 37, 0, 5] = what
        got = ops.sparse_attention(q, bad, vt, index)
        row = got[0, :128, 0]
        if math.isnan(what):
            assert torch.isnan(row).all()
        else:                                                             # the score is q's sign times infinity: NaN, or the key has no weight at all
            up = (q[0, :128, 0, 5] > 0) == (what > 0)
            assert torch.isnan(row[up]).all() and torch.isfinite(row[~up]).all()
        assert torch.equal(got[0, 128:], clean[0, 128:]) and torch.equal(got[0, :, 1:], clean[0, :, 1:])
    bad = q.clone()
    bad[0, 130, 0, 7] = what
    got = ops.sparse_attention(bad, k, vt, index)
    assert torch.isnan(got[0, 130, 0]).all()
    same = torch.ones(Lq, dtype=torch.bool, device="cuda")
    same[130] = False
    assert torch.equal(got[0, same], clean[0, same]) and torch.equal(got[0, 130, 1:], clean[0, 130, 1:])


@pytest.mark.parametrize("Lq", [5, 200])
@pytest.mark.parametrize("what", NANS)
def test_a_value_of_v_that_is_no_number_shows_in_its_column(ops, Lq, what):
    g = gen(77)
    q, k, v = rnd(g, 1, Lq, 2, 128), rnd(g, 1, 640, 2, 128), rnd(g, 1, 640, 2, 128)
    index = torch.tensor([7, 2, 0, 9], dtype=torch.int32, device="cuda").expand(1, 2, (Lq + 127) // 128, 4).contiguous()
    clean = ops.sparse_attention(q, k, vt_of(v), index)
    v[0, 2 * 64 + 11, 1, 50] = what
    v[0, 3 * 64, 0, 9] = what                                             # a block that no list names
    got = ops.sparse_attention(q, k, vt_of(v), index)
    col = got[0, :, 1, 50]
    assert torch.isnan(col).all() if math.isnan(what) else (col == what).all()
    got[0, :, 1, 50] = clean[0, :, 1, 50]
    assert torch.equal(got, clean)
