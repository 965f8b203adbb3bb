"""Soft reads of stored rows against their definitions in 64 bits.

Tolerances.  u is half a step of the operands' type relative to the value, finfo.eps / 2 (bf16 2^-8, fp16 2^-11).  attend: every weight is rounded once to 16 bits before it multiplies its value (u each, so u * sum p |v|
at most), the output once (u |o|); fp32 exponentials and sums add at most 2^-12 of that even over 2^12 keys.  Hence
|o - exact| <= u |exact| + 1.1 u sum p |v| plus what fp16 weights under 2^-14 lose (half a step of 2^-24 a key).
Gradients: grad_v as the output, with p and grad_out; grad_q and grad_k are products of ds, rounded once (u), where
delta comes from the rounded output (u sum |do| |o|, which the sum of absolute terms holds too), with p the fp32 weight.
Hence 2.2 u times the sum of absolute terms.
"""
import math

import pytest

import attention_ref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rand(seed, dtype, *shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def lens(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def check_out(out, lse, ref, dtype, keys):
    want, want_lse, size = ref
    tiny = keys * 2.0 ** -25 * size.amax() if dtype == torch.float16 else 0.0
    tol = unit(dtype) * want.abs() + 1.1 * unit(dtype) * size + tiny + torch.finfo(dtype).smallest_normal * unit(dtype)
    far = ((out.double() - want).abs() - tol)
    assert not torch.isnan(out).any() and far.max().item() <= 0, (far.max().item(), far.argmax().item())
    if lse is not None:
        same = (lse == -math.inf) == (want_lse == -math.inf)
        assert same.all()
        fin = want_lse != -math.inf
        err = (lse.double() - want_lse)[fin].abs()
        # scores of up to 2^6 in fp32 (a few units in their last place), and their exponentials' sum
        assert err.numel() == 0 or (err <= 2e-5 + 1e-6 * want_lse[fin].abs()).all(), err.max().item()


# batch, queries, keys, heads, key heads, width, lengths
SHAPES = [
    (1, 1, 1, 1, 1, 8, None),
    (1, 1, 257, 8, 8, 64, None),
    (2, 3, 0, 4, 2, 64, None),
    (3, 5, 127, 6, 2, 128, (127, 0, 1)),
    (2, 128, 128, 4, 4, 128, None),
    (2, 129, 131, 4, 1, 96, (64, 129)),
    (1, 300, 515, 3, 3, 80, None),
    (4, 1, 1030, 16, 2, 128, (1030, 128, 129, 513)),
    (1, 70, 260, 128, 1, 64, None),
    (2, 257, 640, 10, 2, 72, (640, 385)),
    (1, 33, 4100, 5, 1, 128, None),
    (70, 2, 40, 4, 4, 64, None),
    (1, 1000, 1, 2, 2, 128, None),
]

# large enough for tiles of 128 rows and keys: pairs of row tiles with one range of keys and with several, one row tile with two streams
# of keys, rows that end inside a tile, groups that do not divide one
TILES = [
    (4, 15, 3000, 8, 2, 128, (3000, 129, 2048, 0)),
    (4, 15, 3000, 8, 2, 64, (2999, 1, 700, 3000)),
    (1, 150, 2100, 8, 2, 80, None),
    (2, 333, 1111, 6, 2, 64, (1111, 1000)),
    (2, 333, 1111, 6, 2, 128, (515, 1111)),
    (3, 300, 520, 12, 4, 96, (520, 512, 511)),
    (3, 257, 500, 14, 2, 64, (500, 384, 0)),
    (1, 2048, 384, 4, 4, 128, None),
    (24, 17, 800, 14, 2, 128, None),
    (2, 40, 9000, 3, 1, 8, (9000, 4000)),
    (24, 17, 900, 14, 2, 64, tuple(40 * i for i in range(23)) + (900,)),
    (40, 30, 700, 4, 2, 128, tuple(17 * i for i in range(40))),
    (4, 32, 6000, 8, 2, 64, (6000, 5999, 129, 3000)),
    (4, 32, 6000, 8, 2, 128, (6000, 0, 4481, 3000)),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES + TILES, ids=str)
def test_attend(fm, shape, dtype):
    b, lq, lk, h, hk, d, n = shape
    dt = TYPES[dtype]
    q, k, v = rand(1, dt, b, lq, h, d, scale=1.5), rand(2, dt, b, lk, hk, d), rand(3, dt, b, lk, hk, d)
    n = lens(*n) if n else None
    out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
    check_out(out, lse, R.attend(q, k, v, n), dt, lk)
    assert torch.equal(out, fm.attend(q, k, v, key_lengths=n))
    fm.check_attention_status()


def test_attend_large_scores_and_rising_maxima(fm):
    # keys ordered so that the running maximum rises through the whole sequence, by far more than 2^8 a step
    dt = torch.bfloat16
    q, v = rand(1, dt, 1, 200, 2, 64), rand(3, dt, 1, 1500, 2, 64)
    k = rand(2, dt, 1, 1500, 2, 64) + torch.linspace(-8, 8, 1500, device="cuda", dtype=dt).view(1, -1, 1, 1) * q[:, :1].mean(2, keepdim=True).sign()
    for scale in (0.125, 4.0, 1e-6):
        out, lse = fm.attend(q, k.to(dt), v, scale=scale, return_lse=True)
        want = R.attend(q, k.to(dt), v, scale=scale)
        # scores of a few thousand: fp32 scores are good to 2^-24 of themselves times a few, and so are weights
        top = R.scores(q, k.to(dt), None, scale, False).abs().amax().item()
        assert (lse.double() - want[1]).abs().max() <= 4e-7 * top + 1e-5
        slack = 1 + 2 * top * 2.0 ** -22 / unit(dt)
        assert ((out.double() - want[0]).abs() <= 1.1 * slack * unit(dt) * (want[0].abs() + 2 * want[2]) + 1e-30).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq", [4, 24, 700])
def test_one_key_decides(fm, lq, d):
    """One key's score is far above all others, at every place of a tile in turn, in the first tile and later ones: by less and by more than
    weights may grow before the reference moves, and by more than fp32 exponents reach."""
    dt = torch.bfloat16
    places = torch.arange(0, 600, 1 if lq == 4 else 13, device="cuda")
    b, lk = len(places), 640
    q = torch.zeros(b, lq, 2, d, dtype=dt, device="cuda")
    q[..., 0] = 1
    for jump in (6.0, 14.0, 40.0, 300.0, 30000.0):
        k, v = rand(2, dt, b, lk, 1, d) * 0.25, rand(3, dt, b, lk, 1, d)
        k[torch.arange(b), places, 0, 0] = jump
        out, lse = fm.attend(q, k, v, scale=math.log(2.0), return_lse=True)     # jump is in powers of two
        want = R.attend(q, k, v, scale=math.log(2.0))
        assert ((out.double() - want[0]).abs() <= 2.2 * unit(dt) * want[2] + 1e-6).all(), jump
        assert ((lse.double() - want[1]).abs() <= 2e-5 + 1e-6 * want[1].abs()).all(), jump


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("lq", [4, 700])
def test_nan_in_a_seen_key_comes_through(fm, lq, bad):
    # a NaN or infinite score, wherever it is, makes the row NaN, as the definition does
    dt = torch.float16
    places = torch.arange(0, 300, 7, device="cuda")
    b, lk, d = len(places), 300, 64
    q, k, v = rand(1, dt, b, lq, 1, d).abs() + 0.25, rand(2, dt, b, lk, 1, d), rand(3, dt, b, lk, 1, d)
    k[torch.arange(b), places, 0, 3] = bad
    out, lse = fm.attend(q, k, v, return_lse=True)
    assert torch.isnan(out).all()
    assert (torch.isnan(lse) if math.isnan(bad) else torch.isnan(lse) | (lse == math.inf)).all()


@pytest.mark.parametrize("shape", [(4, 15, 3000, 8, 2, 128), (4, 15, 3000, 8, 2, 64), (2, 333, 1111, 6, 2, 64), (8, 1, 700, 8, 2, 128), (2, 600, 600, 8, 2, 128),
                                   (1, 60, 3000, 2, 2, 128), (24, 40, 800, 14, 2, 128)], ids=str)
def test_results_do_not_depend_on_timing(fm, shape):
    # the same bits again and again, beside other work on the GPU
    b, lq, lk, h, hk, d = shape
    dt = torch.bfloat16
    q, k, v, grad = rand(1, dt, b, lq, h, d), rand(2, dt, b, lk, hk, d), rand(3, dt, b, lk, hk, d), rand(4, dt, b, lq, h, d)
    noise, other = torch.randn(2048, 2048, device="cuda"), torch.cuda.Stream()

    def run():
        out, lse = fm.attend(q, k, v, return_lse=True)
        return (out, lse, *fm.attend_backward(grad, q, k, v, out, lse), fm.attention_mass(q, k, lse))

    want = run()
    for i in range(40):
        with torch.cuda.stream(other):
            for _ in range(i % 5):
                noise @ noise
        for name, x, y in zip(("out", "lse", "grad_q", "grad_k", "grad_v", "mass"), want, run()):
            assert torch.equal(x, y), (name, i)
    # the forward pass alone, many times: tiles that come out of the L2 cache are refilled soon after they are given back
    for i in range(400):
        if i % 3 == 0:
            with torch.cuda.stream(other):
                noise @ noise
        assert torch.equal(want[0], fm.attend(q, k, v)), i
    torch.cuda.synchronize()
    fm.check_attention_status()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lq,lk", [(40, 300), (700, 900)])
def test_attend_masked_rows_have_no_influence(fm, dtype, lq, lk):
    dt = TYPES[dtype]
    q, k, v = rand(1, dt, 3, lq, 4, 64), rand(2, dt, 3, lk, 2, 64), rand(3, dt, 3, lk, 2, 64)
    n = lens(131, 0, lk - 1)
    want = fm.attend(q, k, v, key_lengths=n, return_lse=True)
    bad_k, bad_v = k.clone(), v.clone()
    for i, x in enumerate(n.tolist()):
        bad_k[i, x:], bad_v[i, x:] = math.nan, math.inf
        bad_v[i, x + 1:] = math.nan
    got = fm.attend(q, bad_k, bad_v, key_lengths=n, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert (got[0][1] == 0).all() and (got[1][1] == -math.inf).all()
    grad = rand(4, dt, 3, lq, 4, 64)
    a = fm.attend_backward(grad, q, k, v, *want, key_lengths=n)
    c = fm.attend_backward(grad, q, bad_k, bad_v, *want, key_lengths=n)
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    assert (a[1][1] == 0).all() and (a[2][0, 131:] == 0).all() and (a[0][1] == 0).all()
    m0 = fm.attention_mass(q, k, want[1], key_lengths=n)
    m1 = fm.attention_mass(q, bad_k, want[1], key_lengths=n)
    assert torch.equal(m0, m1) and (m0[1] == 0).all() and (m0[0, :, 131:] == 0).all()


def test_lengths_outside_the_cache_are_clamped(fm):
    dt = torch.float16
    q, k, v = rand(1, dt, 3, 4, 2, 64), rand(2, dt, 3, 100, 2, 64), rand(3, dt, 3, 100, 2, 64)
    out = fm.attend(q, k, v, key_lengths=lens(-5, 1000, 2 ** 31 - 1))
    assert (out[0] == 0).all() and torch.equal(out[1:], fm.attend(q[1:], k[1:], v[1:]))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides(fm, dtype):
    # heads before rows, packed projections, a width cut out of a wider one, repeated sequences and heads
    dt = TYPES[dtype]
    b, lq, lk, h, hk, d = 2, 65, 190, 4, 2, 64
    q = rand(1, dt, b, h, lq, d).permute(0, 2, 1, 3)
    kv = rand(2, dt, b, lk, 2 * hk, d + 8)
    k, v = kv[:, :, 0::2, :d], kv[:, :, 1::2, 8:]
    n = lens(190, 77)
    out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
    check_out(out, lse, R.attend(q, k, v, n), dt, lk)
    dense = fm.attend(q.contiguous(), k.contiguous(), v.contiguous(), key_lengths=n)
    assert torch.equal(out, dense)
    grad = rand(5, dt, h, lq, b, d).permute(2, 1, 0, 3)
    got = fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n)
    want = fm.attend_backward(grad.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), out, lse, key_lengths=n)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert torch.equal(fm.attention_mass(q, k, lse, key_lengths=n),
                       fm.attention_mass(q.contiguous(), k.contiguous(), lse, key_lengths=n))
    one_k, one_v = k[:1].expand(b, -1, -1, -1), v[:, :, :1].expand(-1, -1, hk, -1)
    out, lse = fm.attend(q, one_k, one_v, return_lse=True)
    assert torch.equal(out, fm.attend(q, one_k.contiguous(), one_v.contiguous()))
    got = fm.attend_backward(grad, q, one_k, one_v, out, lse)
    want = fm.attend_backward(grad, q, one_k.contiguous(), one_v.contiguous(), out, lse)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    q1 = q[:, :, :1].expand(-1, -1, h, -1)
    assert torch.equal(fm.attend(q1, k, v), fm.attend(q1.contiguous(), k, v))


def check_grads(got, ref, dtype):
    for name, g, want, size in zip(("q", "k", "v"), got, *ref):
        u = unit(dtype)
        tiny = torch.finfo(dtype).smallest_normal * 2.0 ** -9
        if dtype == torch.float16:
            tiny += 2.0 ** -20 * size.amax()   # fp16 weights and score gradients under 2^-14 of the largest
        far = (g.double() - want).abs() - (u * want.abs() + 2.2 * u * size + tiny)
        assert not torch.isnan(g).any() and far.max().item() <= 0, (name, far.max().item(), far.argmax().item())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [s for s in SHAPES + TILES if s[2]], ids=str)
def test_attend_backward(fm, shape, dtype):
    b, lq, lk, h, hk, d, n = shape
    dt = TYPES[dtype]
    q, k, v = rand(1, dt, b, lq, h, d, scale=1.5), rand(2, dt, b, lk, hk, d), rand(3, dt, b, lk, hk, d)
    grad = rand(4, dt, b, lq, h, d)
    n = lens(*n) if n else None
    out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
    got = fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n)
    check_grads(got, R.backward(grad, q, k, v, n), dt)
    again = fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    fm.check_attention_status()


@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** 10])
def test_backward_of_small_and_large_gradients_in_fp16(fm, size):
    dt = torch.float16
    q, k, v = rand(1, dt, 1, 200, 2, 64, scale=0.25), rand(2, dt, 1, 300, 2, 64), rand(3, dt, 1, 300, 2, 64)
    grad = rand(4, dt, 1, 200, 2, 64)
    # Against the definition on the scaled gradients (comparing with scaled results of the unscaled ones would need a
    # bound for both sides' subnormal steps: half of 2^-24, times the factor).
    grad = (grad.float() * size).to(dt)
    out, lse = fm.attend(q, k, v, return_lse=True)
    check_grads(fm.attend_backward(grad, q, k, v, out, lse), R.backward(grad, q, k, v), dt)


def test_backward_against_differences(fm):
    # the gradient along a direction is the difference quotient of the 64-bit loss
    dt = torch.bfloat16
    q, k, v, grad = (rand(i, dt, 1, 24, 2, 32) for i in range(4))
    out, lse = fm.attend(q, k, v, return_lse=True)
    grads = fm.attend_backward(grad, q, k, v, out, lse)
    for i, g in enumerate(grads):
        step = rand(9 + i, torch.float64, *g.shape)
        e = 1e-5

        def loss(t):
            x = [y.double() for y in (q, k, v)]
            x[i] = x[i] + t * step
            return (R.attend(*x)[0] * grad.double()).sum()

        slope = ((loss(e) - loss(-e)) / (2 * e)).item()
        dot = (g.double() * step).sum().item()
        # every entry is off by 3.2 u of its terms at most; independent signs: a few standard deviations of their sum
        size = R.backward(grad, q, k, v)[1][i]
        assert abs(dot - slope) <= 6 * 3.2 * unit(dt) * (size * step).norm().item()


# batch, new, prefix, own rows, heads, key heads, width, lengths
SHARED = [
    (1, 1, 1, 1, 1, 1, 64, None),
    (5, 3, 1003, 77, 6, 2, 80, (77, 3, 50, 64, 4)),
    (4, 1, 0, 300, 8, 2, 128, (300, 0, 1, 129)),
    (3, 2, 500, 0, 4, 4, 64, None),
    (64, 1, 700, 40, 8, 2, 128, None),
    (33, 4, 260, 140, 16, 2, 96, None),
    (2, 9, 4097, 600, 4, 4, 128, (600, 8)),
    (3, 150, 200, 400, 4, 2, 64, (400, 150, 140)),
    (2, 1, 20000, 5, 8, 1, 128, None),
    (40, 3, 3000, 300, 8, 2, 128, None),
    (40, 3, 3000, 300, 8, 2, 64, tuple(3 + 7 * i for i in range(40))),
    (2, 150, 3000, 2900, 8, 2, 64, (2900, 151)),
    (2, 150, 3000, 2900, 8, 2, 128, (1500, 2900)),
    (3, 200, 1, 1700, 8, 2, 96, (200, 1700, 30)),
    (64, 1, 4000, 1, 32, 4, 72, None),
    (8, 2, 30000, 100, 16, 4, 128, (100, 2, 3, 50, 64, 65, 99, 7)),
    (8, 2, 30000, 100, 16, 4, 64, None),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHARED, ids=str)
def test_attend_shared(fm, shape, dtype):
    b, t, p, s, h, hk, d, n = shape
    dt = TYPES[dtype]
    q, pk, pv = rand(1, dt, b, t, h, d, scale=1.5), rand(2, dt, p, hk, d), rand(3, dt, p, hk, d)
    k, v = rand(4, dt, b, s, hk, d), rand(5, dt, b, s, hk, d)
    n = lens(*n) if n else None
    out, lse = fm.attend_shared(q, pk, pv, k, v, n, return_lse=True)
    check_out(out, lse, R.attend(q, k, v, n, causal=True, shared=(pk, pv)), dt, p + s)
    if n is not None:
        for i, x in enumerate(n.tolist()):
            k[i, x:], v[i, x:] = math.nan, math.nan
        assert torch.equal(out, fm.attend_shared(q, pk, pv, k, v, n))
    fm.check_attention_status()


def test_shared_prefix_equals_copies(fm):
    # the shared prefix gives what every sequence with its own copy of it gives, up to rounding
    dt = torch.bfloat16
    q, pk, pv = rand(1, dt, 3, 1, 8, 64), rand(2, dt, 333, 2, 64), rand(3, dt, 333, 2, 64)
    k, v = rand(4, dt, 3, 50, 2, 64), rand(5, dt, 3, 50, 2, 64)
    n = lens(50, 7, 1)
    out = fm.attend_shared(q, pk, pv, k, v, n)
    copies = [torch.cat([x.expand(3, -1, -1, -1), y], 1) for x, y in ((pk, k), (pv, v))]
    want, _, size = R.attend(q, *copies, lens(383, 340, 334))
    assert ((out.double() - want).abs() <= 2.2 * unit(dt) * size).all()


MASS = SHAPES + [(2, 40, 200, 4, 2, 64, (200, 90)), (1, 513, 700, 8, 2, 128, None), (3, 1, 900, 16, 2, 128, (900, 1, 300))]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", MASS, ids=str)
def test_attention_mass(fm, shape, dtype, causal):
    b, lq, lk, h, hk, d, n = shape
    dt = TYPES[dtype]
    q, k = rand(1, dt, b, lq, h, d, scale=1.5), rand(2, dt, b, lk, hk, d)
    n = lens(*n) if n else None
    lse = R.softmax(R.scores(q, k, n, 1 / math.sqrt(d), causal))[1].permute(0, 2, 1).float().contiguous()
    start = rand(3, torch.float32, b, hk, lk).abs()
    for m in (None, start):
        got = fm.attention_mass(q, k, lse, key_lengths=n, causal=causal, mass=m)
        want = R.mass(q, k, lse, n, causal=causal, start=m)
        # weights are good to a few 2^-22 (fp32 scores of some tens and their exponentials), sums of them to as much
        assert ((got.double() - want).abs() <= 1e-5 * want.abs() + 1e-7).all()
    assert torch.equal(got, fm.attention_mass(q, k, lse, key_lengths=n, causal=causal, mass=start))
    fm.check_attention_status()


EVICT = [
    (1, 1, 1, 8, 1, 0, None),
    (2, 700, 2, 64, 129, 16, (700, 100)),
    (3, 300, 3, 80, 300, 10, None),
    (3, 50, 2, 128, 64, 64, (50, 0, 7)),
    (2, 1000, 1, 256, 1, 1, None),
    (1, 5000, 4, 64, 4999, 0, None),
    (2, 60000, 1, 16, 777, 100, (60000, 50001)),
]


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("shape", EVICT, ids=str)
def test_evict(fm, shape, ties):
    b, lk, hk, d, keep, recent, n = shape
    dt = torch.bfloat16
    k, v = rand(1, dt, b, lk, hk, d), rand(2, dt, b, lk, hk, d)
    m = rand(3, torch.float32, b, hk, lk)
    if ties:
        m = (m * 2).round()
        m[0, 0, ::7] = -0.0
        m[-1, -1, ::11] = math.nan
        m[0, -1, ::13] = math.inf
    n = lens(*n) if n else None
    got = fm.evict(k, v, m, n, keep, recent=recent)
    want = R.evict(k.cpu(), v.cpu(), m.cpu(), n.cpu() if n is not None else None, keep, recent)
    for g, w in zip(got, want):
        assert g.shape == w.shape and g.dtype == w.dtype
        assert torch.equal(torch.nan_to_num(g.cpu(), 7.0), torch.nan_to_num(w, 7.0))


def test_evict_strided(fm):
    dt = torch.float16
    kv = rand(1, dt, 2, 3, 2, 90, 64)                       # heads before rows, keys and values side by side
    k, v = kv[:, :, 0].permute(0, 2, 1, 3), kv[:, :, 1].permute(0, 2, 1, 3)
    m = rand(3, torch.float32, 2, 3, 90).abs()
    got = fm.evict(k, v, m, None, 31, recent=4)
    want = R.evict(k.cpu(), v.cpu(), m.cpu(), None, 31, 4)
    assert all(torch.equal(g.cpu(), w) for g, w in zip(got, want))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("nb,nq,d", [(1, 1, 8), (1000, 3, 64), (5003, 130, 128), (20000, 1, 96)])
def test_index_attend(fm, res, nb, nq, d, dtype):
    dt = TYPES[dtype]
    idx = fm.B200IndexFlat(res, d, fm.METRIC_INNER_PRODUCT, fm.STORAGE_F16 if dtype == "f16" else fm.STORAGE_BF16)
    rows, x = rand(1, dt, nb, d), rand(2, dt, nq, d, scale=1.5)
    values = rand(3, dt, nb, d)
    idx.add(rows.float())
    out, lse = idx.attend(x, values, return_lse=True)
    ref = R.attend(x.view(1, nq, 1, d), rows.view(1, nb, 1, d), values.view(1, nb, 1, d))
    check_out(out.view(1, nq, 1, d), lse.view(1, nq, 1), ref, dt, nb)
    # a growing index: the read before sees the old rows, the one after all of them
    idx.add(rows.float())
    again = idx.attend(x, torch.cat([values, values]))
    assert ((again.double() - ref[0].view(nq, d)).abs() <= 2.5 * unit(dt) * (ref[2].view(nq, d) + ref[0].view(nq, d).abs())
            + (2 * nb * 2.0 ** -25 * ref[2].amax() if dtype == "f16" else 0)).all()
    idx.reset()
    assert (idx.attend(x, values[:0]) == 0).all()
    idx.close()


def test_index_attend_refusals(fm, res):
    idx = fm.B200IndexFlat(res, 64, fm.METRIC_INNER_PRODUCT, fm.STORAGE_F16)
    idx.add(rand(1, torch.float32, 100, 64))
    x, values = rand(2, torch.float16, 4, 64), rand(3, torch.float16, 100, 64)
    for bad in (dict(x=x.bfloat16(), values=values.bfloat16()), dict(x=x, values=values[:99]), dict(x=x[:, :32], values=values),
                dict(x=x.float(), values=values), dict(x=x, values=values.bfloat16())):
        with pytest.raises(ValueError):
            idx.attend(**bad)
    l2 = fm.B200IndexFlat(res, 64, fm.METRIC_L2, fm.STORAGE_F16)
    with pytest.raises(ValueError):
        l2.attend(x, values[:0])
    idx.close()
    l2.close()


def test_a_served_conversation(fm):
    """Prefill, decoding steps behind a shared document, accumulated weights, eviction, and on with the smaller cache."""
    dt = torch.bfloat16
    b, h, hk, d, p, room, keep = 3, 8, 2, 64, 400, 160, 64
    pk, pv = rand(1, dt, p, hk, d), rand(2, dt, p, hk, d)
    k, v = torch.zeros(b, room, hk, d, dtype=dt, device="cuda"), torch.zeros(b, room, hk, d, dtype=dt, device="cuda")
    n = lens(100, 90, 3)
    for i, x in enumerate(n.tolist()):
        k[i, :x], v[i, :x] = rand(10 + i, dt, x, hk, d), rand(20 + i, dt, x, hk, d)
    mass = torch.zeros(b, hk, room, device="cuda")
    want_mass = torch.zeros(b, hk, room, dtype=torch.float64, device="cuda")
    for step in range(4):
        new = 3 if step == 0 else 1
        q = rand(30 + step, dt, b, new, h, d)
        if step:
            at = n.long()
            k[torch.arange(b), at], v[torch.arange(b), at] = rand(40 + step, dt, b, hk, d), rand(50 + step, dt, b, hk, d)
            n = n + 1
        out, lse = fm.attend_shared(q, pk, pv, k, v, n, return_lse=True)
        check_out(out, lse, R.attend(q, k, v, n, causal=True, shared=(pk, pv)), dt, p + room)
        mass = fm.attention_mass(q, k, lse, key_lengths=n, causal=True, mass=mass)
        want_mass = R.mass(q, k, lse, n, causal=True, start=want_mass)
        assert ((mass.double() - want_mass).abs() <= 1e-5 * want_mass + 1e-6).all()
    nk, nv, nm, rows, nn = fm.evict(k, v, mass, n, keep, recent=8)
    ref = R.evict(k.cpu(), v.cpu(), mass.cpu(), n.cpu(), keep, 8)
    assert all(torch.equal(g.cpu(), w) for g, w in zip((nk, nv, nm, rows, nn), ref))
    q = rand(60, dt, b, 1, h, d)
    out, lse = fm.attend_shared(q, pk, pv, nk, nv, nn, return_lse=True)
    check_out(out, lse, R.attend(q, nk, nv, nn, causal=True, shared=(pk, pv)), dt, p + keep)
    # the prefix's own weights: all queries as one sequence
    m = fm.attention_mass(q.reshape(1, b, h, d), pk.unsqueeze(0), lse.reshape(1, b, h))
    total = m.sum((0, 2)) + fm.attention_mass(q, nk, lse, key_lengths=nn, causal=True).sum((0, 2))
    assert torch.allclose(total.cpu(), torch.full((hk,), float(b * h // hk)), rtol=1e-4)


def test_streams_and_graphs(fm):
    dt = torch.float16
    q, k, v = rand(1, dt, 2, 130, 4, 64), rand(2, dt, 2, 900, 2, 64), rand(3, dt, 2, 900, 2, 64)
    pk, pv, grad = rand(4, dt, 3000, 2, 64), rand(5, dt, 3000, 2, 64), rand(6, dt, 2, 130, 4, 64)
    n = lens(900, 411)

    def run():
        out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
        grads = fm.attend_backward(grad, q, k, v, out, lse, key_lengths=n)
        m = fm.attention_mass(q, k, lse, key_lengths=n)
        return (out, lse, *grads, m, *fm.attend_shared(q[:, :1], pk, pv, k, v, n, return_lse=True), *fm.evict(k, v, m, n, 100, recent=9))

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, other))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    n.copy_(lens(17, 899))
    fresh = run()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(x, y) for x, y in zip(fresh, o))
    a, c = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):                                     # both at once
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(c):
            graphs[1].replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(x, y) for x, y in zip(fresh, o))
    fm.check_attention_status()


def test_offsets_beyond_32_bits(fm):
    # a cache of 4.3 GB: the last rows lie behind 2^32 bytes, the last sequence behind 2^31 elements
    dt = torch.bfloat16
    lk, hk, d = 1_100_000, 8, 128
    k = torch.zeros(2, lk, hk, d, dtype=dt, device="cuda")
    v = torch.zeros(2, lk, hk, d, dtype=dt, device="cuda")
    q = rand(1, dt, 2, 1, hk, d)
    tail = 300
    k[:, -tail:] = rand(2, dt, 2, tail, hk, d) * 3
    v[:, -tail:] = rand(3, dt, 2, tail, hk, d)
    out, lse = fm.attend(q, k, v, return_lse=True, scale=1.0)
    s = torch.einsum("bhd,bjhd->bhj", q[:, 0].double(), k[:, -tail:].double())
    e = torch.exp(s)
    total = e.sum(-1) + (lk - tail)
    want = torch.einsum("bhj,bjhd->bhd", e, v[:, -tail:].double()) / total.unsqueeze(-1)
    size = torch.einsum("bhj,bjhd->bhd", e, v[:, -tail:].double().abs()) / total.unsqueeze(-1)
    assert ((out[:, 0].double() - want).abs() <= 3 * unit(dt) * size + 1e-12).all()
    assert (lse[:, 0].double() - torch.log(total)).abs().max() < 1e-4
    m = fm.attention_mass(q, k, lse, scale=1.0)
    w = e / total.unsqueeze(-1)
    assert ((m[:, :, -tail:].double() - w).abs() <= 2e-4 * w + 1e-9).all()
    got = fm.evict(k, v, m, None, 400, recent=50)
    assert torch.equal(got[3][:, :, -50:].cpu(), torch.arange(lk - 50, lk, dtype=torch.int32).expand(2, hk, 50))
    live = got[3].permute(0, 2, 1).long()
    assert torch.equal(got[0], torch.gather(k, 1, live.unsqueeze(-1).expand(-1, -1, -1, d)))


def test_refusals(fm):
    dt = torch.float16
    q, k, v = rand(1, dt, 2, 4, 4, 64), rand(2, dt, 2, 9, 2, 64), rand(3, dt, 2, 9, 2, 64)
    n = lens(9, 4)
    bad = [
        dict(q=q.float(), k=k, v=v), dict(q=q, k=k.bfloat16(), v=v), dict(q=q, k=k, v=v[:, :8]), dict(q=q, k=k[:1], v=v[:1]),
        dict(q=q[:, :, :3], k=k, v=v), dict(q=q[..., :60], k=k[..., :60], v=v[..., :60]), dict(q=q[0], k=k, v=v),
        dict(q=q, k=k, v=v, key_lengths=n.long()), dict(q=q, k=k, v=v, key_lengths=n[:1]), dict(q=q, k=k, v=v, scale=0.0),
        dict(q=q, k=k, v=v, scale=math.inf), dict(q=q, k=k, v=v, scale=math.nan), dict(q=q, k=k.cpu(), v=v),
        dict(q=q, k=k[:, :1].expand(-1, 9, -1, -1), v=v), dict(q=q.transpose(1, 3).contiguous().transpose(1, 3), k=k, v=v),
        dict(q=q, k=k, v=v, key_lengths=n.cpu()),
    ]
    wide = rand(4, dt, 2, 4, 4, 136)
    bad.append(dict(q=wide, k=wide[:, :, :2], v=wide[:, :, :2]))
    odd = rand(4, dt, 2 * 9 * 2 * 64 + 1)[1:].view(2, 9, 2, 64)                 # off the 16-byte boundary
    bad.append(dict(q=q, k=odd, v=v))
    skew = rand(4, dt, 2, 9, 2, 68)[..., :64]                                   # strides of 68 elements
    bad.append(dict(q=q, k=skew, v=v))
    for args in bad:
        with pytest.raises(ValueError):
            fm.attend(**args)
    with pytest.raises(TypeError):
        fm.attend(q.cpu().numpy(), k, v)
    out, lse = fm.attend(q, k, v, return_lse=True)
    grad = torch.ones_like(out)
    for args in (dict(grad_out=grad[:, :3]), dict(lse=lse.half()), dict(lse=lse.transpose(1, 2)), dict(out=out[:, :3]),
                 dict(grad_out=torch.ones((), dtype=dt, device="cuda").expand(2, 4, 4, 64))):
        with pytest.raises(ValueError):
            fm.attend_backward(**{**dict(grad_out=grad, q=q, k=k, v=v, out=out, lse=lse), **args})
    m = torch.zeros(2, 2, 9, device="cuda")
    for args in (dict(mass=m[:, :1]), dict(mass=m.double()), dict(lse=lse[:1])):
        with pytest.raises(ValueError):
            fm.attention_mass(**{**dict(q=q, k=k, lse=lse), **args})
    for args in (dict(keep=0), dict(keep=3, recent=4), dict(keep=3, recent=-1), dict(keep=3, mass=m[:, :, :8])):
        with pytest.raises(ValueError):
            fm.evict(**{**dict(k=k, v=v, mass=m, key_lengths=n), **args})
    with pytest.raises(ValueError):
        fm.attend(q.clone().requires_grad_(), k, v)
    with torch.no_grad():
        fm.attend(q.clone().requires_grad_(), k, v)


def test_nothing_to_do(fm):
    dt = torch.bfloat16
    e = torch.empty
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        q = e(*shape, dtype=dt, device="cuda")
        k = torch.ones(shape[0], 5, 2, 64, dtype=dt, device="cuda")
        out, lse = fm.attend(q, k, k, return_lse=True)
        assert out.shape == shape and lse.shape == shape[:3]
        gq, gk, gv = fm.attend_backward(q, q, k, k, out, lse)
        assert gq.shape == shape and (gk == 0).all() and (gv == 0).all() and gk.shape == k.shape
        assert (fm.attention_mass(q, k, lse) == 0).all()
    q = torch.ones(2, 3, 2, 64, dtype=dt, device="cuda")
    k = e(2, 0, 2, 64, dtype=dt, device="cuda")
    out, lse = fm.attend(q, k, k, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    gq, gk, gv = fm.attend_backward(q, q, k, k, out, lse)
    assert (gq == 0).all() and gk.shape == k.shape
    assert fm.attention_mass(q, k, lse).shape == (2, 2, 0)
    nk, nv, nm, rows, n = fm.evict(k, k, e(2, 2, 0, device="cuda"), None, 4)
    assert (nk == 0).all() and (rows == -1).all() and (n == 0).all() and (nm == 0).all()


def test_neither_queries_nor_keys(fm):
    q, k = (torch.empty(2, 0, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    out, lse = fm.attend(q, k, k, return_lse=True)
    assert [x.shape for x in fm.attend_backward(q, q, k, k, out, lse)] == [q.shape, k.shape, k.shape]
    assert fm.attention_mass(q, k, lse).shape == (2, 2, 0)


def test_options_given_as_tensors_are_read_at_every_call(fm):
    dt = torch.float16
    q, k, v = rand(1, dt, 1, 5, 2, 64), rand(2, dt, 1, 40, 2, 64), rand(3, dt, 1, 40, 2, 64)
    m = rand(4, torch.float32, 1, 2, 40)
    scale, keep = torch.tensor(0.5), torch.tensor(8)
    for s, n in ((0.5, 8), (0.125, 5)):
        scale.fill_(s)
        keep.fill_(n)
        assert torch.equal(fm.attend(q, k, v, scale=scale), fm.attend(q, k, v, scale=s))
        assert fm.evict(k, v, m, None, keep)[0].shape[1] == n


def test_scales_up_to_the_largest(fm):
    dt = torch.float16
    q = torch.zeros(1, 20, 1, 64, dtype=dt, device="cuda")
    v = rand(3, dt, 1, 300, 1, 64)
    for n in (20, 300):                                     # scores of 0, whatever the scale
        out = fm.attend(q, torch.ones_like(v[:, :n]), v[:, :n], scale=2e38)
        assert torch.equal(out, fm.attend(q, torch.ones_like(v[:, :n]), v[:, :n], scale=1.0))
    with pytest.raises(ValueError):
        fm.attend(q, v, v, scale=2.5e38)


@pytest.mark.parametrize("shape", [(64, 1, 5000, 700, 32, 8, 128), (128, 1, 4096, 512, 16, 2, 64), (33, 2, 9000, 60, 8, 2, 96)], ids=str)
def test_prefix_and_own_rows_at_the_same_time(fm, shape):
    b, t, p, n, h, hk, d = shape
    dt = torch.bfloat16
    q, pk, pv = rand(1, dt, b, t, h, d, scale=1.5), rand(2, dt, p, hk, d), rand(3, dt, p, hk, d)
    k, v = rand(4, dt, b, n, hk, d), rand(5, dt, b, n, hk, d)
    length = torch.randint(0, n + 1, (b,), generator=torch.Generator().manual_seed(6)).int().cuda()
    out, lse = fm.attend_shared(q, pk, pv, k, v, length, return_lse=True)
    check_out(out, lse, R.attend(q, k, v, length, causal=True, shared=(pk, pv)), dt, p + n)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = fm.attend_shared(q, pk, pv, k, v, length) + 0       # read at once by a kernel that is launched plainly
    for _ in range(100):
        assert torch.equal(fm.attend_shared(q, pk, pv, k, v, length), out)
        g.replay()
        assert torch.equal(captured, out)
    fm.check_attention_status()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_reader_is_trained(fm, dtype):
    """attend and attend_backward as the two halves of an autograd function, under eager calls and side streams."""
    dt = TYPES[dtype]

    class Read(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, n):
            out, lse = fm.attend(q, k, v, key_lengths=n, return_lse=True)
            ctx.save_for_backward(q, k, v, n, out, lse)
            return out

        @staticmethod
        def backward(ctx, grad):
            q, k, v, n, out, lse = ctx.saved_tensors
            return (*fm.attend_backward(grad.contiguous(), q, k, v, out, lse, key_lengths=n), None)

    q, k, v = (rand(i, dt, *s).requires_grad_() for i, s in ((1, (2, 140, 4, 64)), (2, (2, 333, 2, 64)), (3, (2, 333, 2, 64))))
    n, w = lens(333, 65), rand(4, dt, 2, 140, 4, 64)
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            (Read.apply(q, k, v, n) * w).sum().backward()
        torch.cuda.current_stream().wait_stream(stream)
        check_grads([x.grad for x in (q, k, v)], R.backward(w, q.detach(), k.detach(), v.detach(), n), dt)
        for x in (q, k, v):
            x.grad = None
    fm.check_attention_status()
