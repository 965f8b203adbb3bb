"""Soft reads at the edges of their ranges.  u is half a step of the operands' type relative to the value."""
import math

import pytest

import attention_ref as R
from test_gpu_attention import TYPES, check_grads, check_out, lens, rand, unit

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


# ---- empty sides -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lq,lk", [(0, 2000), (2000, 0), (0, 100_000), (3000, 0)])
def test_gradient_of_a_call_with_an_empty_side(fm, lq, lk, dtype):
    # long enough that the streamed rows, were there any, would be cut into ranges
    q, k, v = (torch.ones(2, n, h, 64, dtype=TYPES[dtype], device="cuda") for n, h in ((lq, 4), (lk, 2), (lk, 2)))
    out, lse = fm.attend(q, k, v, return_lse=True)
    gq, gk, gv = fm.attend_backward(q, q, k, v, out, lse)
    assert gq.shape == q.shape and gk.shape == k.shape and gv.shape == v.shape
    assert (gq == 0).all() and (gk == 0).all() and (gv == 0).all()
    fm.check_attention_status()


# ---- fp16 gradients far below the largest --------------------------------------------------------


def far_from_rows(got, grad, q, k, v, n=None, scale=None):
    """How far fp16 gradients are beyond their bounds, entry by entry (at most 0 when within), every entry judged by its own terms.

    A term's score gradient (or weight) is rounded once: u of it, uniform at worst, u / sqrt(3) in the mean square; with independent
    signs a sum of such errors stays within 4.5 u (almost eight standard deviations) of the root of the terms' squares.  delta comes from the rounded
    output: u of sum |do| |o|.  The result is rounded once: u, at least 2^-25.  A multiplication by a power of two leaves the bound 2 |do| max |v| of a row's score gradients
    between 2^12 and 2^14 (and a weight of 1 at 2^12): what lies below fp16's normal range then errs by 2^-25 / 2^12 of that bound.  For
    grad_k a row's query entries take the inverse factors, the largest of them kept at 2^-3 or more, which lets the smallest err by 2^-22 of it; rows so far below the call's largest that this
    limit holds them err by 2^-53 of that.  fp32 sums: 2^-23 of their running value a step of 16 terms, in ranges of 16,384 at most."""
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    seen = R.visible(n, b, lq, lk, False, q.device).any(1)
    k, v = R.live(k, seen), R.live(v, seen)
    p, _ = R.softmax(R.scores(q, k, n, scale, False))
    g, qq, kk, vv = (R.heads_first(x, h) for x in (grad, q, k, v))                     # [b, h, rows, d]
    o = p @ vv
    ds = p * (g @ vv.transpose(-1, -2) - (g * o).sum(-1, keepdim=True)) * scale
    dabs = (g.abs() * o.abs()).sum(-1, keepdim=True) * scale
    bound = 2 * g.norm(dim=-1, keepdim=True) * vv.norm(dim=-1).amax(-1).view(b, h, 1, 1) * scale
    qmax, kmax = qq.abs().amax(-1, keepdim=True), kk.abs().amax((-1, -2), keepdim=True)
    largest = (bound * qmax).view(b, hk, -1).amax(-1)

    def keys(x):                                                                       # sums over a group
        return x.view(b, hk, h // hk, lk, -1).sum(2).permute(0, 2, 1, 3)

    def turned(x):
        return x.transpose(-1, -2)

    u, rows = unit(torch.float16), lq * h // hk
    want = ((ds @ kk).permute(0, 2, 1, 3), keys(turned(ds) @ qq), keys(turned(p) @ g))
    sig = ((ds.square() @ kk.square()).sqrt().permute(0, 2, 1, 3), keys(turned(ds.square()) @ qq.square()).sqrt(),
           keys(turned(p.square()) @ g.square()).sqrt())
    extra = ((u * dabs * (p @ kk).abs() + 4.5 * lk ** 0.5 * 2.0 ** -37 * bound * kmax).permute(0, 2, 1, 3),
             4.5 * u * keys(turned((p * dabs).square()) @ qq.square()).sqrt()
             + 4.5 * 2.0 ** -37 * (bound * qmax).square().view(b, hk, -1).sum(-1).sqrt().view(b, 1, hk, 1)
             + rows * 2.0 ** -53 * largest.view(b, 1, hk, 1) + 2.0 ** -22 * keys(turned(ds.abs()) @ qmax),
             4.5 * 2.0 ** -37 * g.square().amax(-1).view(b, hk, -1).sum(-1).sqrt().view(b, 1, hk, 1))
    far = []
    for x, w, s, e, terms in zip(got, want, sig, extra, (lk, rows, rows)):
        assert not torch.isnan(x).any()
        far.append(((x.double() - w).abs() - (u * w.abs() + 4.5 * u * s + e + 2.0 ** -25
                                              + min(terms, 16384) / 16 * 2.0 ** -23 * (w.abs() + 4.5 * s))).max().item())
    return far


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk", [(256, 4096), (100, 1531)])
@pytest.mark.parametrize("low,high", [(0, 8), (0, 12), (-4, 14), (-10, 5), (-14, 14)])
def test_rows_of_small_and_large_gradients_together(fm, lq, lk, d, low, high):
    """One row's output gradient is 2^(high - low) times the others'.  It reads one key alone, so that the other keys' gradients
    come from the other rows only."""
    dt = torch.float16
    q, k, v = rand(1, dt, 1, lq, 2, d), rand(2, dt, 1, lk, 2, d), rand(3, dt, 1, lk, 2, d)
    grad = (rand(4, torch.float32, 1, lq, 2, d) * 2.0 ** low).to(dt)
    grad[0, 17] = 0
    grad[0, 17, :, 5] = 2.0 ** high
    q[0, 17], k[0, 40] = 0, 0
    q[0, 17, :, 3], k[0, 40, :, 3] = 64, 8 * math.sqrt(d) / 4       # score 128 at key 40; the others' are below 32
    k[0, :40, :, 3].clamp_(max=1)
    k[0, 41:, :, 3].clamp_(max=1)
    out, lse = fm.attend(q, k, v, return_lse=True)
    got = fm.attend_backward(grad, q, k, v, out, lse)
    far = far_from_rows(got, grad, q, k, v)
    assert max(far) <= 0, far
    fm.check_attention_status()


@pytest.mark.parametrize("lq,lk,h,hk", [(64, 1000, 4, 2), (300, 3000, 6, 2), (5, 1500, 96, 1)])
def test_rows_of_every_magnitude(fm, lq, lk, h, hk):
    # output gradients and queries over 2^20 and 2^12, in turn
    dt = torch.float16
    q, k, v = rand(1, torch.float32, 2, lq, h, 64), rand(2, dt, 2, lk, hk, 64), rand(3, dt, 2, lk, hk, 64)
    grad = rand(4, torch.float32, 2, lq, h, 64)
    r = torch.arange(2 * lq * h, device="cuda").view(2, lq, h, 1)
    q = (q * 2.0 ** (-(r * 7 % 13).float())).to(dt)
    grad = (grad * 2.0 ** ((r * 11 % 21).float() - 10)).to(dt)
    n = lens(lk, lk // 3)
    out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
    far = far_from_rows(fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n), grad, q, k, v, n)
    assert max(far) <= 0, far


@pytest.mark.parametrize("lq,lk", [(32, 1_000_000), (200, 100_000)])
def test_fp16_gradients_over_many_keys(fm, lq, lk):
    # a weight is about 1 / keys
    dt = torch.float16
    q, k, v, grad = rand(1, dt, 1, lq, 1, 64), rand(2, dt, 1, lk, 1, 64), rand(3, dt, 1, lk, 1, 64), rand(4, dt, 1, lq, 1, 64)
    grad = grad * 16
    out, lse = fm.attend(q, k, v, return_lse=True)
    far = far_from_rows(fm.attend_backward(grad, q, k, v, out, lse), grad, q, k, v)
    assert max(far) <= 0, far


def test_fp16_gradients_of_large_values(fm):
    # value rows of a norm up to 160,000, all in line with the output gradient
    dt = torch.float16
    q, k = rand(1, dt, 1, 150, 2, 64) * 0.125, rand(2, dt, 1, 200, 2, 64) * 0.125
    v = torch.where(torch.arange(200, device="cuda").view(1, 200, 1, 1) % 2 == 0, 20000.0, -20000.0).expand(1, 200, 2, 64).to(dt).contiguous()
    grad = torch.full((1, 150, 2, 64), 2.0 ** -7, dtype=dt, device="cuda")
    for n in (None, lens(2)):
        out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
        far = far_from_rows(fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n), grad, q, k, v, n)
        assert max(far) <= 0, far


def test_fp16_gradients_keep_to_their_sequence_and_key_head(fm):
    # what other sequences and key heads hold changes no bit, nor do rows behind the end
    dt = torch.float16
    q, k, v, grad = rand(1, dt, 2, 90, 4, 64), rand(2, dt, 2, 400, 2, 64), rand(3, dt, 2, 400, 2, 64), rand(4, dt, 2, 90, 4, 64)
    n = lens(400, 333)

    def run(q, k, v, grad):
        out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
        return fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n)

    want = run(q, k, v, grad)
    other = [x.clone() for x in (q, k, v, grad)]
    other[3][0] *= 2.0 ** 11
    other[2][0] *= 2.0 ** 9
    other[0][0] *= 2.0 ** 3
    other[1][1, 333:], other[2][1, 333:] = math.nan, 60000.0
    got = run(*other)
    assert all(torch.equal(x[1], y[1]) for x, y in zip(want, got))
    other = [x.clone() for x in (q, k, v, grad)]
    other[3][:, :, :2] *= 2.0 ** 11
    other[2][:, :, 0] = math.inf
    got = run(*other)
    assert torch.equal(want[0][:, :, 2:], got[0][:, :, 2:])
    assert all(torch.equal(want[i][:, :, 1], got[i][:, :, 1]) for i in (1, 2))


def test_fp16_gradients_of_zero_and_of_rows_that_are_not_finite(fm):
    dt = torch.float16
    q, k, v, grad = rand(1, dt, 1, 90, 2, 64), rand(2, dt, 1, 400, 2, 64), rand(3, dt, 1, 400, 2, 64), rand(4, dt, 1, 90, 2, 64)
    q[0, 3], grad[0, 5] = 0, 0
    out, lse = fm.attend(q, k, v, return_lse=True)
    got = fm.attend_backward(grad, q, k, v, out, lse)
    assert max(far_from_rows(got, grad, q, k, v)) <= 0 and (got[0][0, 5] == 0).all()
    zero = fm.attend_backward(torch.zeros_like(grad), q, k, v, out, lse)
    assert all((x == 0).all() for x in zero)
    bad = grad.clone()
    bad[0, 7, 1, 2] = math.inf
    gq, gk, gv = fm.attend_backward(bad, q, k, v, out, lse)
    assert torch.isnan(gq[0, 7, 1]).any() and torch.isnan(gk[:, :, 1]).any() and (torch.isnan(gv[:, :, 1, 2]) | (gv[:, :, 1, 2] == math.inf)).all()
    keep = torch.arange(90, device="cuda") != 7
    far = far_from_rows((gq[:, keep][:, :, 0:1].contiguous(), got[1][:, :, :1], got[2][:, :, :1]), grad[:, keep][:, :, :1], q[:, keep][:, :, :1], k[:, :, :1], v[:, :, :1])
    assert far[0] <= 0
    assert torch.equal(gk[:, :, 0], got[1][:, :, 0]) and torch.equal(gv[:, :, 0], got[2][:, :, 0])
    # the row's NaN does not reach other rows' query gradients
    far = far_from_rows((gq[:, keep][:, :, 1:].contiguous(), got[1][:, :, 1:], got[2][:, :, 1:]), grad[:, keep][:, :, 1:], q[:, keep][:, :, 1:], k[:, :, 1:], v[:, :, 1:])
    assert far[0] <= 0


# ---- weights far below a row's largest -------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,lq,lk", [(75, 256, 1_000_000), (1200, 1, 300_000)])
def test_a_long_tail_of_small_weights(fm, b, lq, lk, d, dtype):
    """One key's score lies 18 above all others': each of these weighs 2^-26 of it, all together 0.5 % to 1.5 %, and the sequences are so many that
    a row's keys are one range.  In fp16 the largest weight is held at 2^7 or more and a weight below the type's normal range errs by 2^-25 at
    most, a key 2^-32 of the largest value."""
    dt = TYPES[dtype]
    q = torch.zeros(b, lq, 1, d, dtype=dt, device="cuda")
    q[..., 0] = 1
    k = torch.zeros(1, lk, 1, d, dtype=dt, device="cuda")
    v = rand(3, dt, 1, lk, 1, d) * 0.25 + 1
    top = 12_345
    k[0, top, 0, 0] = 18
    v[0, top] = 0.25
    out, lse = fm.attend(q, k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), scale=1.0, return_lse=True)
    w = torch.full((lk, 1), math.exp(-18.0), dtype=torch.float64, device="cuda")
    w[top] = 1
    total = w.sum()
    vv = v[0, :, 0].double()
    want, size = (w * vv).sum(0) / total, (w * vv.abs()).sum(0) / total
    tol = unit(dt) * want.abs() + 1.1 * unit(dt) * size + lk * 2.0 ** -32 * vv.abs().max()
    # sums in the tensor cores are of 2^15 terms, each of which loses 2^-25 of the sum at most
    tol = tol + 2.0 ** -10 * size
    assert ((out.double() - want).abs() <= tol).all(), ((out.double() - want).abs() / want.abs()).max().item()
    assert ((lse.double() - (18 + torch.log(total))).abs() <= 1e-4 + lk / 32 * 2.0 ** -24).all()
    fm.check_attention_status()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("b,lq,lk,d", [(80, 130, 70_000, 64), (80, 130, 70_000, 128), (80, 300, 40_000, 72), (74, 100, 140_000, 64), (74, 60, 140_000, 128)])
def test_sums_of_long_ranges(fm, b, lq, lk, d, dtype):
    # more keys a range than are summed up in one go; the largest score rises all the way; ends at and beside the borders
    dt = TYPES[dtype]
    q, v = rand(1, dt, b, lq, 1, d), rand(3, dt, 1, lk, 1, d)
    k = rand(2, dt, 1, lk, 1, d) * 0.5
    q[..., 0] = 1
    k[0, :, 0, 0] = torch.linspace(-6, 6, lk, device="cuda") * math.sqrt(d)
    ends = [lk, 32768, 32769, 65536, 0, 32767, 65537, lk - 1]
    n = torch.tensor([min(lk, ends[i % len(ends)]) for i in range(b)], dtype=torch.int32, device="cuda")
    out, lse = fm.attend(q, k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), key_lengths=n, return_lse=True)
    for i in range(8):
        check_out(out[i:i + 1], lse[i:i + 1], R.attend(q[i:i + 1], k, v, n[i:i + 1]), dt, lk)
    assert torch.equal(out[8:16, :5], fm.attend(q, k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), key_lengths=n)[8:16, :5])
    fm.check_attention_status()


# ---- scales near the end of fp32's range -----------------------------------------------------------


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("place", [5, 200])
@pytest.mark.parametrize("lq,lk", [(4, 300), (700, 300), (700, 1200)])
def test_scores_near_the_end_of_fp32(fm, lq, lk, place, dtype):
    """Scores that leave fp32's range when they are scaled count as infinite: a row with a positive one is NaN, negative ones weigh nothing.
    Those that stay inside give the row that the definition gives."""
    dt = TYPES[dtype]
    q = torch.zeros(1, lq, 1, 64, dtype=dt, device="cuda")
    k, v = torch.zeros(1, lk, 1, 64, dtype=dt, device="cuda"), rand(3, dt, 1, lk, 1, 64)
    k[0, place, 0, 0] = 2
    for i, x in enumerate((0.0, 1.0, -1.0, 0.5)):            # scores of 0, 4e38, -4e38 and 2e38 at that key, of 0 elsewhere
        q[0, i::4, 0, 0] = x
    out, lse = fm.attend(q, k, v, scale=2e38, return_lse=True)
    vv = v[0, :, 0].double()
    rest = torch.arange(lk, device="cuda") != place
    u = unit(dt)

    def near(x, want, values):
        # equal weights that are powers of two at most: products and sums are exact but for fp32's rounding, the output is rounded once
        return ((x.double() - want).abs() <= u * want.abs() + lk * 2.0 ** -23 * values.abs().mean(0) + 2.0 ** -25).all()

    assert near(out[0, 0::4, 0], vv.mean(0), vv)
    assert ((lse[0, 0::4] - math.log(lk)).abs() < 1e-4).all()
    assert torch.isnan(out[0, 1::4]).all()
    assert (torch.isnan(lse[0, 1::4]) | (lse[0, 1::4] == math.inf)).all()
    assert near(out[0, 2::4, 0], vv[rest].mean(0), vv)
    assert ((lse[0, 2::4] - math.log(lk - 1)).abs() < 1e-4).all()
    assert near(out[0, 3::4, 0], vv[place], vv[place:place + 1])
    assert ((lse[0, 3::4] / 2e38 - 1).abs() < 1e-5).all()
    fm.check_attention_status()


@pytest.mark.parametrize("lq", [4, 700])
def test_keys_whose_scores_are_minus_infinity(fm, lq):
    # every score of the first row is -4e38, of the second -4e38 up to the last key, whose score is 0
    dt = torch.bfloat16
    q = torch.zeros(1, lq, 1, 64, dtype=dt, device="cuda")
    q[0, 0::2, 0, 0], q[0, 1::2, 0, 1] = -1, -1
    k, v = torch.zeros(1, 500, 1, 64, dtype=dt, device="cuda"), rand(3, dt, 1, 500, 1, 64)
    k[..., :2] = 2
    k[0, -1, 0, 1] = 0
    out, lse = fm.attend(q, k, v, scale=2e38, return_lse=True)
    assert (out[0, 0::2] == 0).all() and (lse[0, 0::2] == -math.inf).all()
    assert (out[0, 1::2, 0] == v[0, -1, 0]).all() and (lse[0, 1::2].abs() < 1e-5).all()
    fm.check_attention_status()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("b,t,p,n,h,hk,d", [(300, 1, 300_000, 40, 16, 2, 64), (300, 1, 300_000, 40, 16, 2, 128), (40, 300, 0, 70_000, 2, 1, 64),
                                            (40, 300, 70_000, 40_000, 2, 1, 128)])
def test_sums_of_long_prefixes_and_prompts(fm, b, t, p, n, h, hk, d, dtype):
    dt = TYPES[dtype]
    q, pk, pv = rand(1, dt, b, t, h, d, scale=1.5), rand(2, dt, p, hk, d), rand(3, dt, p, hk, d)
    k, v = rand(4, dt, 1, n, hk, d).expand(b, -1, -1, -1), rand(5, dt, 1, n, hk, d).expand(b, -1, -1, -1)
    length = torch.tensor([max(n - 37 * i, t) for i in range(b)], dtype=torch.int32, device="cuda")
    out, lse = fm.attend_shared(q, pk, pv, k, v, length, return_lse=True)
    for i in (0, 1, b - 1):
        one = slice(i, i + 1)
        check_out(out[one], lse[one], R.attend(q[one], k[one], v[one], length[one], causal=True, shared=(pk, pv)), dt, p + n)
    assert torch.equal(out, fm.attend_shared(q, pk, pv, k, v, length))
    fm.check_attention_status()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_sums_of_many_queries_in_the_gradient(fm, dtype):
    """One query's weight times its output gradient is 64 at key 0; 500,000 others give 1.8e-6 each, 0.9 together: just below 2^-25 of the sum."""
    dt = TYPES[dtype]
    b, lq, lk, d = 110, 500_000, 128, 64                     # so many sequences that the queries are one range
    q = torch.zeros(1, lq, 1, d, dtype=dt, device="cuda")
    q[..., 0] = 1
    q[0, 0, 0, 0] = -8
    k, v = torch.zeros(1, lk, 1, d, dtype=dt, device="cuda"), rand(3, dt, 1, lk, 1, d)
    k[0, 0, 0, 0] = -8.375
    grad = torch.ones(1, lq, 1, d, dtype=dt, device="cuda")
    grad[0, 0] = 64
    many = (lambda x: x.expand(b, -1, -1, -1))
    out, lse = fm.attend(many(q), many(k), many(v), scale=1.0, return_lse=True)
    gv = fm.attend_backward(many(grad), many(q), many(k), many(v), out, lse, scale=1.0)[2]
    p0 = 1 / (1 + 127 * math.exp(-67))
    want = 64 * p0 + (lq - 1) * math.exp(-8.375) / (127 + math.exp(-8.375))
    # weights and the result are rounded once, sums of 2^15 terms lose 2^-25 a term
    assert ((gv[:, 0].double() / want - 1).abs() <= 2.2 * unit(dt) + 2.0 ** -10).all(), (gv[0, 0, 0, 0].item(), want)
    assert (gv == gv[:1]).all()
    fm.check_attention_status()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lq", [128, 100])
def test_sums_of_many_keys_in_the_gradient(fm, lq, dtype):
    """Key 0 has half of a row's weight, 2^19 others the rest: their score gradients, -1 / 2^19 of its own each, meet key entries of 7/16
    where it has 64, and are less than 2^-25 of the sum."""
    dt = TYPES[dtype]
    b, lk, d = 110, 2 ** 19 + 1, 64
    q = torch.zeros(b, lq, 1, d, dtype=dt, device="cuda")
    q[..., 0] = 1
    k, v = torch.full((1, lk, 1, d), 0.4375, dtype=dt, device="cuda"), torch.zeros(1, lk, 1, d, dtype=dt, device="cuda")
    k[..., 0] = 0
    k[0, 0] = 64
    k[0, 0, 0, 0] = 13.1875                                  # ln 2^19 = 13.17
    v[0, 0] = 1
    many = (lambda x: x.expand(b, -1, -1, -1))
    top = k[0, 0, 0, 0].item()
    grad = torch.ones_like(q)
    out, lse = fm.attend(q, many(k), many(v), scale=1.0, return_lse=True)
    gq = fm.attend_backward(grad, q, many(k), many(v), out, lse, scale=1.0)[0]
    p0 = math.exp(top) / (math.exp(top) + lk - 1)
    ds = p0 * (1 - p0) * d
    want = ds * (64 - 0.4375)
    # score gradients are rounded once, delta comes from the rounded output: u p0 d, of which key 0 and all others take their weights; the
    # result is rounded once; sums of 2^15 terms lose 2^-25 a term
    u = unit(dt)
    tol = u * want + 1.1 * u * ds * 64.4375 + u * p0 * d * (p0 * 64 + (1 - p0) * 0.4375) + 2.0 ** -10 * ds * 64
    assert ((gq[..., 1:].double() - want).abs() <= tol).all(), (gq[0, 0, 0, 1].item(), want, tol)
    fm.check_attention_status()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("b,lq,lk,h,d", [(40, 33_000, 200, 3, 64), (3, 100, 70_000, 8, 72), (40, 40, 70_000, 3, 128), (1, 70_000, 100, 2, 128)])
def test_gradients_of_long_ranges(fm, b, lq, lk, h, d, dtype):
    # sums that are moved to memory on the way, in one range and in several, against the definition
    dt = TYPES[dtype]
    q, k, v = rand(1, dt, b, lq, h, d, scale=1.5), rand(2, dt, b, lk, 1, d), rand(3, dt, b, lk, 1, d)
    grad = rand(4, dt, b, lq, h, d)
    n = torch.tensor([max(lk - 1000 * (i % 3), lk // 2) for i in range(b)], dtype=torch.int32, device="cuda")
    out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
    got = fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n)
    for i in {0, 1 % b, b - 1}:
        one = slice(i, i + 1)
        check_grads([x[one] for x in got], R.backward(grad[one], q[one], k[one], v[one], n[one]), dt)
    again = fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    fm.check_attention_status()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_log_sums_of_a_million_keys(fm, dtype):
    """The weights of 1,000,000 equal keys, 1.5 % of the first one's all together, are added up with fp32's rounding: 96 or 32 at once, in chains of
    2^15 keys (half a step of 2^-23 each, 512 of them) that are then added up (31), and exponentials are good to 2.7e-6."""
    dt = TYPES[dtype]
    b, lk = 75, 1_000_000
    q = torch.zeros(b, 256, 1, 64, dtype=dt, device="cuda")
    q[..., 0] = 1
    k = torch.zeros(1, lk, 1, 64, dtype=dt, device="cuda")
    k[0, 0, 0, 0] = 18
    many = (lambda x: x.expand(b, -1, -1, -1))
    lse = fm.attend(q, many(k), many(k), scale=1.0, return_lse=True)[1]
    want = 18 + math.log1p((lk - 1) * math.exp(-18.0))
    # 18 itself is held to 2^-20
    assert (lse.double() - want).abs().max() <= (512 + 31) * 2.0 ** -24 + 2.7e-6 + 2.0 ** -20 * 2


# ---- groups of odd size ----------------------------------------------------------------------------


GROUPS = [(2, 3, 300, 65, 1, 64, (300, 77)), (1, 5, 1000, 96, 1, 128, None), (2, 1, 4000, 127, 1, 72, (4000, 1)), (1, 40, 513, 200, 2, 64, None),
          (3, 70, 140, 34, 2, 128, (140, 0, 129)), (1, 300, 200, 65, 1, 64, None)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", GROUPS, ids=str)
def test_groups_that_do_not_fill_their_tiles(fm, shape, dtype):
    # 65 to 127 heads a key head: a gradient tile of 64 and one that is part empty; 17, 100: a queries' tile with rows left over
    b, lq, lk, h, hk, d, n = shape
    dt = TYPES[dtype]
    q, k, v = rand(1, dt, b, lq, h, d, scale=1.5), rand(2, dt, b, lk, hk, d), rand(3, dt, b, lk, hk, d)
    grad = rand(4, dt, b, lq, h, d)
    n = lens(*n) if n else None
    out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
    check_out(out, lse, R.attend(q, k, v, n), dt, lk)
    check_grads(fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n), R.backward(grad, q, k, v, n), dt)
    for causal in (False, True):
        row = R.softmax(R.scores(q, k, n, 1 / math.sqrt(d), causal))[1].permute(0, 2, 1).float().contiguous()
        got, want = fm.attention_mass(q, k, row, key_lengths=n, causal=causal), R.mass(q, k, row, n, causal=causal)
        assert ((got.double() - want).abs() <= 1e-5 * want.abs() + 1e-7).all()
    pk, pv = rand(5, dt, 333, hk, d), rand(6, dt, 333, hk, d)
    out, lse = fm.attend_shared(q, pk, pv, k, v, n, return_lse=True)
    check_out(out, lse, R.attend(q, k, v, n, causal=True, shared=(pk, pv)), dt, 333 + lk)
    fm.check_attention_status()


# ---- eviction --------------------------------------------------------------------------------------


def test_evicted_rows_and_rows_behind_the_end_do_not_come_through(fm):
    # NaN and infinities in rows behind the end, and in rows that are evicted, reach nothing; in rows that stay they come through
    dt = torch.float16
    b, lk, hk, d, keep = 3, 500, 2, 64, 40
    k, v = rand(1, dt, b, lk, hk, d), rand(2, dt, b, lk, hk, d)
    m = rand(3, torch.float32, b, hk, lk).abs() + 0.5
    n = lens(500, 300, 17)
    want = fm.evict(k, v, m, n, keep, recent=5)
    kept = torch.zeros(b, hk, lk + 1, dtype=torch.bool, device="cuda").scatter_(2, want[3].long() % (lk + 1), True)[..., :lk]
    gone = ~kept.permute(0, 2, 1)
    k2, v2, m2 = k.clone(), v.clone(), m.clone()
    k2[gone], v2[gone] = math.nan, math.inf
    for i, x in enumerate(n.tolist()):
        m2[i, :, x:] = math.nan
        m2[i, 0, x:] = math.inf
    got = fm.evict(k2, v2, m2, n, keep, recent=5)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    k2 = k.clone()
    k2[0, -1] = math.nan                                     # among the recent ones
    assert torch.isnan(fm.evict(k2, v, m, n, keep, recent=5)[0][0, keep - 1]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("scale", [1.0, 3e3, 7e5, 1e8, 3e12, 1e20, 1e30, 1e37])
@pytest.mark.parametrize("lq,lk", [(4, 300), (700, 300), (700, 1200), (60, 9000)])
def test_ties_of_large_scores(fm, lq, lk, scale, dtype):
    """Keys of equal score, whatever its size, share a row: at the end of a rise, in different tiles, warps and ranges.  Scores are products of two
    numbers, exact in fp32; the next lower one lies a sixteenth below."""
    dt = TYPES[dtype]
    a, c = (torch.tensor(x, dtype=dt).item() for x in (1.1, 0.7))
    q = torch.zeros(1, lq, 1, 64, dtype=dt, device="cuda")
    q[..., 0] = a
    q[0, 1::2] *= -1
    k, v = torch.zeros(1, lk, 1, 64, dtype=dt, device="cuda"), rand(3, dt, 1, lk, 1, 64)
    k[..., 0] = torch.linspace(-0.9, 0.9, lk, device="cuda").to(dt).clamp(-c + c / 16, c - c / 16).view(1, lk, 1)
    ties = torch.tensor([3, 17, 40, 129, 200, lk // 2, lk - 20, lk - 1], device="cuda").unique()
    k[0, ties, 0, 0] = c
    lows = torch.tensor([2, 30, 131, lk // 2 + 1, lk - 3], device="cuda").unique()
    k[0, lows, 0, 0] = -c
    out, lse = fm.attend(q, k, v, scale=scale, return_lse=True)
    # with the maximum taken off first: at 1e20 a 64-bit log-sum does not hold the number of ties any more
    s = R.scores(q, k, None, scale, False)
    p, vv = torch.softmax(s, -1), R.heads_first(v, 1)
    want, size, want_lse = (p @ vv).permute(0, 2, 1, 3), (p @ vv.abs()).permute(0, 2, 1, 3), torch.logsumexp(s, -1).permute(0, 2, 1)
    u = unit(dt)
    # scores are held to 2^-24 of themselves where tiles, warps and ranges meet; beyond 2^13 only equal ones share a row
    near = min(abs(a * c * scale) * 2.0 ** -22, 0.0 if a * c * scale / 16 > 30 else 1.0)
    assert ((out.double() - want).abs() <= u * want.abs() + (1.1 * u + near + 3e-6) * size + 2.0 ** -24).all()
    assert ((lse.double() - want_lse).abs() <= 1e-6 * want_lse.abs() + 2e-5).all()
    fm.check_attention_status()


# ---- accumulated weights of every number of rows in a tile ------------------------------------------


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lq,h,hk", [(12, 8, 2), (49, 2, 2), (13, 8, 2), (16, 16, 4), (97, 1, 1), (1, 128, 1), (32, 8, 2)])
def test_accumulated_weights_of_wide_rows(fm, lq, h, hk, dtype):
    # 48 to 128 packed rows of d = 128 over many key tiles: the rings of three and of two
    dt = TYPES[dtype]
    b, lk, d = 3, 3333, 128
    q, k, n = rand(1, dt, b, lq, h, d, scale=1.5), rand(2, dt, b, lk, hk, d), lens(3333, 1024, 129)
    for causal in (False, True):
        lse = R.softmax(R.scores(q, k, n, 1 / math.sqrt(d), causal))[1].permute(0, 2, 1).float().contiguous()
        got, want = fm.attention_mass(q, k, lse, key_lengths=n, causal=causal), R.mass(q, k, lse, n, causal=causal)
        assert ((got.double() - want).abs() <= 1e-5 * want.abs() + 1e-7).all()
        assert torch.equal(got, fm.attention_mass(q, k, lse, key_lengths=n, causal=causal))
    fm.check_attention_status()
