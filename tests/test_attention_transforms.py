"""The soft reads record no derivatives and have no batching rules: tensors that ask for them are refused, before anything else about them is
looked at, so that this needs no GPU."""
import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad  # noqa: E402


def tensors():
    x = torch.ones(1, 2, 2, 64, dtype=torch.float16)
    return x, x[0], torch.ones(1, 2, 2), torch.ones(1, 2, 2)


def calls(fm, x):
    _, shared, lse, mass = tensors()
    plain = tensors()[0]
    return [lambda: fm.attend(plain, x, plain), lambda: fm.attend_shared(x, shared, shared, plain, plain),
            lambda: fm.attend_backward(x, plain, plain, plain, plain, lse), lambda: fm.attention_mass(plain, x, lse),
            lambda: fm.evict(plain, x, mass, None, 1)]


@pytest.mark.parametrize("gradients", [True, False])
@pytest.mark.parametrize("which", range(5))
def test_tangents_are_refused(fm, which, gradients):
    x = tensors()[0]
    with forward_ad.dual_level(), torch.set_grad_enabled(gradients):
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="tangent"):
            calls(fm, dual)[which]()
        with pytest.raises(ValueError, match="CUDA"):       # tensors without one go on to the ordinary checks
            calls(fm, x)[which]()


def test_tangent_of_log_sums(fm):
    x, _, lse, _ = tensors()
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            fm.attention_mass(x, x, forward_ad.make_dual(lse, lse))


@pytest.mark.parametrize("which", range(5))
def test_transforms_are_refused(fm, which):
    x = tensors()[0]

    def run(y):
        calls(fm, y)[which]()
        return (y * 2).sum()

    for transform in (lambda: torch.func.vmap(run)(torch.stack([x, x])), lambda: torch.func.jvp(run, (x,), (x,)),
                      lambda: torch.func.grad(run)(x)):
        with pytest.raises(ValueError, match="torch.func"):
            transform()


def test_other_tensors_inside_a_transform(fm):
    x = tensors()[0]

    def run(y):
        with pytest.raises(ValueError, match="CUDA"):       # not wrapped: an ordinary call
            fm.attend(x, x, x)
        return (y * 2).sum()

    torch.func.grad(run)(torch.ones(3))


def test_an_autograd_function_under_forward_mode(fm):
    # torch strips the tangents before its forward: nothing to refuse there
    seen = []

    class F(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            with pytest.raises(ValueError, match="CUDA"):
                fm.attend(x, x, x)
            seen.append(1)
            return x * 2

        @staticmethod
        def jvp(ctx, t):
            return t * 2

    x = tensors()[0]
    with forward_ad.dual_level():
        F.apply(forward_ad.make_dual(x, x))
    assert seen
